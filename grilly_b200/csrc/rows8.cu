// Rows in 8 bits: quantise, read back, RMSNorm with the residual's addition into 8-bit rows, and that norm's backward
// pass from the 8-bit checkpoint of its input. The definitions stand with the entry points in include/grilly_b200.h.
//
// All of them are bound by HBM. A persistent CTA of 512 threads per SM works on several rows at a time, a team of 16 to 512
// threads on each (32 values per thread). Every team has a ring of rows in shared memory that bulk copies fill several rows
// ahead, so that memory is read all the time and not only while a block has nothing else to do (blocks that each load,
// reduce and store a row reached half the bandwidth). A row goes from there into registers, is reduced once and written once.
// Rows that start off 16-byte boundaries (odd lengths) are copied from the boundary below and shifted into place as they are
// read (load_piece); 16-bit and 32-bit results leave in the vectors that memory has, 8-bit rows start on boundaries always.
// 16384 x 4096 bf16: the norm with both outputs 91 us (5.9 TB/s), its backward pass with the residual's gradient 85 us
// (5.5 TB/s), quantise 39 us (5.1 TB/s), read back 35 us (5.8 TB/s); a plain copy runs at 6.5 TB/s.
// 16384 x 4001 bf16: 131 us (4.0 TB/s), 132 (3.5), 52 (3.8) and 36 (5.5); fp32: 196 us (4.7), 185 (4.6), 68 (4.8). The
// shifts are the difference: half of the issue slots are used, by 36 % (norm) and 55 % (backward) more
// instructions than for aligned rows. Read and stored value by value the same took 177, 146, 79 and 59 us in bf16; only
// fp32's backward pass was faster, 171.
#include "rows8.h"
#include "rows8_sum.cuh"
#include "ptx.cuh"
#include "f32x2.cuh"
#include <cuda_bf16.h>
#include <algorithm>
#include <initializer_list>

namespace gb {
namespace {

constexpr int PER_THREAD = 32;         // values of a row per thread
constexpr int CTA = 512;
constexpr int MIN_TEAM = 16;
constexpr int MAX_TEAMS = CTA / MIN_TEAM;
constexpr int MAX_DEPTH = 8;           // rows in a team's ring
constexpr uint32_t FULL = 0xffffffffu;
constexpr uint32_t INF_BITS = 0x7f800000u;
#define ROWS8_NAN __uint_as_float(0x7fffffffu)

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
// of magnitudes: non-negative floats order like their bits, an infinity is above every finite number and a NaN above that
__device__ __forceinline__ float warp_max(float v) { return __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(v))); }
__device__ __forceinline__ bool not_finite(float magnitude) { return __float_as_uint(magnitude) >= INF_BITS; }

// A piece of a row, as a thread holds it in pairs: VEC neighbouring values (16 bytes of T) from a column that is a multiple
// of VEC, wherever the row starts in memory.
template <int VEC>
struct Piece {
  static constexpr int PAIRS = VEC / 2;
  F2 v[PAIRS];
};
__device__ __forceinline__ void load_vec(const float* p, Piece<4>& x) {
  const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(p);
  x.v[0].v = t.x;
  x.v[1].v = t.y;
}
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, Piece<8>& x) {
  const uint4 t = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x.v[i] = F2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void store_vec(float* p, const Piece<4>& x) { *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(x.v[0].v, x.v[1].v); }
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const Piece<8>& x) {
  *reinterpret_cast<uint4*>(p) = make_uint4(x.v[0].bf16(), x.v[1].bf16(), x.v[2].bf16(), x.v[3].bf16());
}
__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void from_words(const uint32_t* w, Piece<4>& x) {
  x.v[0] = F2(__uint_as_float(w[0]), __uint_as_float(w[1]));
  x.v[1] = F2(__uint_as_float(w[2]), __uint_as_float(w[3]));
}
__device__ __forceinline__ void from_words(const uint32_t* w, Piece<8>& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x.v[i] = F2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
// The piece at column c of a row of F values (0 past its end) in shared memory. ODD: rows are not on 16-byte boundaries;
// the row starts `off` bytes behind `row`. Two vectors then hold the piece, and what belongs to it is shifted out of them:
// by words with two selections, by half a word with a funnel shift, the same for all threads. (Values read one by one
// took twice as long: two thirds of the instructions of a kernel were loads and conversions.)
template <bool ODD, int VEC, class T>
__device__ __forceinline__ void load_piece(const uint8_t* row, int off, int c, int F, Piece<VEC>& x) {
  const uint8_t* p = row + c * sizeof(T);
  if constexpr (!ODD) {
    load_vec(reinterpret_cast<const T*>(p), x);
  } else {
    uint32_t w[6];
    if constexpr (sizeof(T) == 4) {
      const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 16);
      const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 5; ++k) w[k] = off & 8 ? v[k + 2] : v[k];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = off & 4 ? w[k + 1] : w[k];
    } else {
      const uint2* p8 = reinterpret_cast<const uint2*>(p + (off & 8));
      const uint2 a = p8[0], b = p8[1], d = p8[2];
      const uint32_t v[6] = {a.x, a.y, b.x, b.y, d.x, d.y};
#pragma unroll
      for (int k = 0; k < 5; ++k) w[k] = off & 4 ? v[k + 1] : v[k];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], (off & 2) * 8);
    }
    if (c + VEC > F) {
      constexpr int PER_WORD = 4 / sizeof(T);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int left = F - c - k * PER_WORD;
        if (left <= 0) w[k] = 0;
        else if (left < PER_WORD) w[k] &= 0xffffu;
      }
    }
    from_words(w, x);
  }
}
// Writes a piece to its place in such a row, in shared memory.
__device__ __forceinline__ void place_piece(uint8_t* row, int off, int c, const Piece<4>& x) {
  uint32_t* p = reinterpret_cast<uint32_t*>(row + off + c * 4);
  float f[4];
  x.v[0].get(f[0], f[1]);
  x.v[1].get(f[2], f[3]);
  if (off & 4) {
    p[0] = __float_as_uint(f[0]);
    *reinterpret_cast<F2*>(p + 1) = F2(f[1], f[2]);
    p[3] = __float_as_uint(f[3]);
  } else {
    *reinterpret_cast<F2*>(p) = x.v[0];
    *reinterpret_cast<F2*>(p + 2) = x.v[1];
  }
}
__device__ __forceinline__ void place_piece(uint8_t* row, int off, int c, const Piece<8>& x) {
  uint8_t* p = row + off + c * 2;
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = x.v[k].bf16();
  if (off & 2) {
    *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint32_t*>(p + 2 + 4 * k) = __funnelshift_r(w[k], w[k + 1], 16);
    *reinterpret_cast<uint16_t*>(p + 14) = static_cast<uint16_t>(w[3] >> 16);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t*>(p + 4 * k) = w[k];
  }
}
// Stores the 16 bytes of a row (F values at `row` in memory, which lies `off` bytes behind a boundary) that start `at` bytes
// behind that boundary; at the row's ends only what belongs to it.
template <class T>
__device__ __forceinline__ void store_between(T* row, int off, int at, int F, uint4 x) {
  const int from = at - off, end = F * static_cast<int>(sizeof(T));
  uint8_t* p = reinterpret_cast<uint8_t*>(row) + from;
  if (from >= 0 && from + 16 <= end) {
    *reinterpret_cast<uint4*>(p) = x;
  } else {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 16; k += sizeof(T)) {
      if (from + k < 0 || from + k >= end) continue;
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p + k) = w[k / 4];
      else *reinterpret_cast<uint16_t*>(p + k) = static_cast<uint16_t>(w[k / 4] >> (k % 4 * 8));
    }
  }
}
// The sums of 16 bytes of values, each rounded to T. (Of two bf16 numbers the sum rounded once is the fp32 sum rounded to
// bf16: where the fp32 sum is not exact, the smaller one is too small to move the larger.)
template <class T>
__device__ __forceinline__ uint4 add16(uint4 a, uint4 b) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  uint32_t s[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      s[k] = __float_as_uint(__uint_as_float(x[k]) + __uint_as_float(y[k]));
    } else {
      const __nv_bfloat162 t = __hadd2_rn(*reinterpret_cast<const __nv_bfloat162*>(&x[k]), *reinterpret_cast<const __nv_bfloat162*>(&y[k]));
      s[k] = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
  return make_uint4(s[0], s[1], s[2], s[3]);
}
// Gamma in shared memory: as it is, or for pieces of 8 first every piece's first four values, then every piece's last four
// (neighbouring lanes then read neighbouring 16 bytes instead of every second 16).
template <int VEC>
__device__ __forceinline__ int gamma_at(int col, int F) {
  return VEC == 8 ? ((col >> 2) & 1) * ((F + 7) / 8 * 4) + (col >> 3) * 4 + (col & 3) : col;
}
// the columns' fp32 parameters (1 where there are none)
template <int VEC>
__device__ __forceinline__ void load_gamma(const float* gamma, int c, int F, Piece<VEC>& g) {
  if (!gamma) {
#pragma unroll
    for (int j = 0; j < Piece<VEC>::PAIRS; ++j) g.v[j] = F2(1.f, 1.f);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(gamma + gamma_at<VEC>(c + j, F));
      g.v[j / 2].v = t.x;
      g.v[j / 2 + 1].v = t.y;
    }
  }
}

// max(amax / 127, 2^-126) or NaN. The quotient is the product with the rounded 1 / 127 and one correction by its remainder
// (Markstein), the correctly rounded one for every finite amax that is not clamped (checked over all significands).
__device__ __forceinline__ float row_scale(float a) {
  const float r = 1.f / 127.f, q = a * r;
  return not_finite(a) ? ROWS8_NAN : fmaxf(fmaf(fmaf(-127.f, q, a), r, q), ROWS8_TINY);
}
// q is 127 x / a rounded to the nearest integer (ties to even), a the row's largest |x|: the quotient by the scale before
// the scale's own rounding. Ties are common where the values lie on a coarse grid, x = a / 2 for one, and a product with
// one float falls to either side of them.
struct RowInverse {
  float hi, lo;
};
struct RowInverse2 {
  F2 hi, lo;
  __device__ __forceinline__ explicit RowInverse2(RowInverse r) : hi(r.hi, r.hi), lo(r.lo, r.lo) {}
};
// ONE = false: 127 / a as a sum of two floats. A product and a fused multiply-add give the quotient right to 2^-47 before
// its rounding to fp32, so that a tie comes out as that tie (and what is nearer to one than 2^-18, half a step of an fp32
// number of 64 to 127, becomes one).
// ONE: for bf16 values one float rounded up and one fused multiply-add do. 254 x and a (2 k + 1) have 16 bits each and are
// equal or 2^-16 apart, equal only where a is 127 * 2^j (the inverse is a power of two then, the product exact) or
// x = a / 2, and that tie goes up, to 64.
// scale: a / 127 or, for a of at most 127 * 2^-126, 2^-126, whose inverse is exact. No division: it would stand between a
// row's reduction and its stores (quantise 44 us with it, 40 without, at 16384 x 4096 bf16).
template <bool ONE>
__device__ __forceinline__ RowInverse row_inverse(float scale, float a) {
  const float t = __fdividef(1.f, scale), d = t * (1.f / 127.f);   // t to 2 ulp; scales lie in [2^-126, 2^121]
  const float rest = a > 127.f * ROWS8_TINY ? fmaf(-a, t, 127.f) : 0.f;
  if (!ONE) return {t, rest * d};
  const float hi = fmaf(rest, d, t);                               // to half an ulp; exact where 127 / a is a power of two
  return {rest != 0.f && fmaf(-a, hi, 127.f) > 0.f ? fmaf(hi, 0x1p-23f, hi) : hi, 0.f};
}
constexpr float MAGIC = 12582912.f;   // 1.5 * 2^23: the sum has no fraction bits, and the integer is in its low byte
template <bool ONE>
__device__ __forceinline__ F2 quotient2(F2 x, const RowInverse2& inv) {
  const F2 magic(MAGIC, MAGIC);
  return ONE ? fma2(x, inv.hi, magic) : add2(fma2(x, inv.hi, mul2(x, inv.lo)), magic);
}
// Four bytes come out of three byte permutes; conversions would run at a quarter rate.
template <bool ONE>
__device__ __forceinline__ uint32_t round4(F2 a, F2 b, const RowInverse2& inv) {
  float f[4];
  quotient2<ONE>(a, inv).get(f[0], f[1]);
  quotient2<ONE>(b, inv).get(f[2], f[3]);
  return __byte_perm(__byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x0040),
                     __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x0040), 0x5410);
}
// keep: all ones, or zero for a row that is not finite.
template <bool ONE>
__device__ __forceinline__ int8_t round1(float x, RowInverse inv, uint32_t keep) {
  return static_cast<int8_t>(__float_as_uint(ONE ? fmaf(x, inv.hi, MAGIC) : __fadd_rn(fmaf(x, inv.hi, __fmul_rn(x, inv.lo)), MAGIC)) & keep);
}
// (8-bit rows start on 16-byte boundaries and have room for whole pieces)
template <bool ONE, int VEC>
__device__ __forceinline__ void store_q(int8_t* row, int c, const Piece<VEC>& x, const RowInverse2& inv, uint32_t keep) {
  const uint32_t w = round4<ONE>(x.v[0], x.v[1], inv) & keep;
  if constexpr (VEC == 8) *reinterpret_cast<uint2*>(row + c) = make_uint2(w, round4<ONE>(x.v[2], x.v[3], inv) & keep);
  else *reinterpret_cast<uint32_t*>(row + c) = w;
}
// four signed bytes as floats: byte + 128 below the bits of 2^23, then the offset taken off; exact
__device__ __forceinline__ void unpack4(uint32_t w, F2& lo, F2& hi) {
  w ^= 0x80808080u;
  const F2 offset(-8388736.f, -8388736.f);
  lo = add2(F2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441))), offset);
  hi = add2(F2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443))), offset);
}
template <int VEC>
__device__ __forceinline__ void load_q(const uint8_t* row, int c, Piece<VEC>& x) {
  if constexpr (VEC == 8) {
    const uint2 t = *reinterpret_cast<const uint2*>(row + c);
    unpack4(t.x, x.v[0], x.v[1]);
    unpack4(t.y, x.v[2], x.v[3]);
  } else {
    unpack4(*reinterpret_cast<const uint32_t*>(row + c), x.v[0], x.v[1]);
  }
}

// ---- the ring
// Up to three row tensors (all 16-byte aligned) and the geometry that the host chose.
struct Ring {
  const void* src[3];
  long long pitch[3];        // bytes from row to row in memory
  long long total[3];        // bytes of the tensor
  int bytes[3];              // bytes of one row
  int at[3];                 // where a tensor's row lies in a slot
  int tensors, slot;         // slot: bytes, a multiple of 16
  int aligned;               // every row starts on a 16-byte boundary and holds a multiple of 16 bytes
  int depth;                 // slots per team
  int gamma_at, slots_at;    // offsets in shared memory: barriers first, then reductions, gamma, slots
  long long rows;
  long long first_tail;      // from this row on, bytes past the tensors' last 16-byte boundary are needed
  int F;
  int* err;
};
struct RowStats {
  float sq, my, mh;            // sum of squares, max |h gamma|, max |h|
};
constexpr int RED_AT = MAX_TEAMS * MAX_DEPTH * 8;              // RowStats [2][CTA / 32]
constexpr int ABORT_AT = RED_AT + 2 * (CTA / 32) * 12;
constexpr int GAMMA_AT = (ABORT_AT + 4 + 15) / 16 * 16;

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// A team's view of the ring (TEAM threads). All of a team's threads call next() and done() together.
template <int TEAM>
struct Team {
  static constexpr int TEAMS = CTA / TEAM;
  const Ring& g;
  uint8_t* smem;
  uint64_t* bars;
  volatile int* abort_flag;
  int team, tid, slot, parity;   // parity: of the slot's barrier
  int ok;                        // whether the row's wait ended; the team's word on it after agree()
  uint32_t flip;                 // which half of the reduction scratch
  long long row, step;

  __device__ __forceinline__ Team(const Ring& ring, uint8_t* shared) : g(ring), smem(shared), flip(0) {
    team = threadIdx.x / TEAM;
    tid = threadIdx.x % TEAM;
    bars = reinterpret_cast<uint64_t*>(smem) + team * g.depth;
    abort_flag = reinterpret_cast<volatile int*>(smem + ABORT_AT);
    row = static_cast<long long>(team) * gridDim.x + blockIdx.x;
    step = static_cast<long long>(TEAMS) * gridDim.x;
    slot = 0;
    parity = 0;
  }
  // whole CTA: barriers, gamma, the first rows on their way
  template <int VEC>
  __device__ void start(const float* gamma) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < TEAMS * g.depth; ++i) mbar_init(reinterpret_cast<uint64_t*>(smem) + i, 1);
      *abort_flag = 0;
      fence_mbar_init();
    }
    __syncthreads();
    if (tid == 0) {
      for (int d = 0; d < g.depth; ++d) fetch(row + d * step, d);
    }
    float* gm = reinterpret_cast<float*>(smem + g.gamma_at);
    if (gamma)
      for (int c = threadIdx.x; c < (g.F + VEC - 1) / VEC * VEC; c += CTA) gm[gamma_at<VEC>(c, g.F)] = c < g.F ? __ldg(gamma + c) : 0.f;
    __syncthreads();
  }
  // the team's lanes of its warp (a team of 16: half a warp)
  __device__ __forceinline__ uint32_t lanes() const { return TEAM >= 32 ? FULL : 0xffffu << (threadIdx.x & 16); }
  // the aligned bytes [from, to) of row r of tensor i that a copy brings, relative to the tensor
  __device__ void span(int i, long long r, long long& from, long long& to) const {
    from = r * g.pitch[i] & ~15ll;
    to = min((r * g.pitch[i] + g.bytes[i] + 15) & ~15ll, g.total[i] & ~15ll);
    if (to < from) to = from;
  }
  __device__ uint8_t* slot_of(int d) const { return smem + g.slots_at + (team * g.depth + d) * g.slot; }
  __device__ void fetch(long long r, int d) const {
    if (r >= g.rows) return;
    if (g.aligned) {
      uint8_t* to = slot_of(d);
      mbar_expect_tx(&bars[d], g.slot);
      bulk_load(to, static_cast<const uint8_t*>(g.src[0]) + r * g.pitch[0], g.bytes[0], &bars[d]);
      if (g.tensors > 1) bulk_load(to + g.at[1], static_cast<const uint8_t*>(g.src[1]) + r * g.pitch[1], g.bytes[1], &bars[d]);
      if (g.tensors > 2) bulk_load(to + g.at[2], static_cast<const uint8_t*>(g.src[2]) + r * g.pitch[2], g.bytes[2], &bars[d]);
      return;
    }
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
    if constexpr (TEAM <= 32) __syncwarp(lanes());
    else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TEAM) : "memory");
  }
  // Waits for the current row. Whether the wait ended (else it is reported and the team stops) is agreed on at once and
  // returned, or, LATER, by the reduction that follows: one barrier less.
  template <bool LATER>
  __device__ bool next() {
    ok = mbar_wait(&bars[slot], static_cast<uint32_t>(parity), abort_flag) ? 1 : 0;
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
    if (row >= g.first_tail) sync();
    if (!LATER) agree();
    return LATER || ok != 0;
  }
  // a barrier of the team at which ok becomes that of all
  __device__ void agree() {
    if constexpr (TEAM <= 32) {
      ok = __all_sync(lanes(), ok);
    } else {
      asm volatile(
          "{\n\t"
          ".reg .pred p, q;\n\t"
          "setp.ne.s32 p, %1, 0;\n\t"
          "bar.red.and.pred q, %2, %3, p;\n\t"
          "selp.s32 %0, 1, 0, q;\n\t"
          "}\n"
          : "=r"(ok) : "r"(ok), "r"(team + 1), "n"(TEAM) : "memory");
    }
  }
  // the current row of tensor i, from the 16-byte boundary at or before its first value, and that value's distance
  __device__ uint8_t* bytes(int i) const { return slot_of(slot) + g.at[i]; }
  __device__ int off(int i) const { return static_cast<int>(row * g.pitch[i] & 15); }
  // everything of the row has been read. WROTE: its slot was written to as well, before a bulk copy fills it
  template <bool WROTE>
  __device__ void done() {
    sync();
    if (tid == 0) {
      if (WROTE) fence_proxy_async_smem();
      fetch(row + g.depth * step, slot);
    }
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
  // over the team, in an order that its size alone decides; a point where the team agrees on ok
  template <bool kSum, bool kMax, bool kTwo>
  __device__ RowStats reduce(RowStats s) {
    if constexpr (TEAM <= 32) agree();
    if constexpr (TEAM == 16) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        if constexpr (kSum) s.sq += __shfl_xor_sync(lanes(), s.sq, o);
        if constexpr (kMax) s.mh = max_abs(s.mh, __shfl_xor_sync(lanes(), s.mh, o), 0.f);
        if constexpr (kTwo) s.my = max_abs(s.my, __shfl_xor_sync(lanes(), s.my, o), 0.f);
      }
      return s;
    }
    if constexpr (kSum) s.sq = warp_sum(s.sq);
    if constexpr (kMax) s.mh = warp_max(s.mh);
    if constexpr (kTwo) s.my = warp_max(s.my);
    if constexpr (TEAM > 32) {
      constexpr int WARPS = TEAM / 32;
      const int lane = threadIdx.x & 31;
      RowStats* red = reinterpret_cast<RowStats*>(smem + RED_AT) + flip * (CTA / 32);
      flip ^= 1;             // the other half is free again once every thread has passed this row's barriers
      if (lane == 0) red[threadIdx.x >> 5] = s;
      agree();
      s = lane < WARPS ? red[team * WARPS + lane] : RowStats{0.f, 0.f, 0.f};
      if constexpr (kSum) s.sq = warp_sum(s.sq);
      if constexpr (kMax) s.mh = warp_max(s.mh);
      if constexpr (kTwo) s.my = warp_max(s.my);
    }
    return s;
  }
};
// The pieces of a row that a thread has: i counts them, c is the first column. Rows shorter than a team's full width leave
// the loop for all threads at once.
#define FOR_PIECES(i, c)                                                                       \
  _Pragma("unroll") for (int i = 0, c = t.tid * VEC; i < NV; ++i, c += TEAM * VEC) \
    if (i * TEAM * VEC >= F) break;                                              \
    else if (c < F)

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
template <class T, int TEAM, bool ODD>
__global__ void __launch_bounds__(CTA, 1) quantize_rows_kernel(const __grid_constant__ Ring ring, int8_t* q, float* scale, long long ld) {
  constexpr int VEC = 16 / sizeof(T), NV = PER_THREAD / VEC, PAIRS = Piece<VEC>::PAIRS;
  extern __shared__ __align__(16) uint8_t smem[];
  Team<TEAM> t(ring, smem);
  t.template start<VEC>(nullptr);
  const int F = ring.F;
  for (; t.row < ring.rows; t.template done<false>()) {
    t.template next<true>();
    const uint8_t* xp = t.bytes(0);
    const int off = ODD ? t.off(0) : 0;
    Piece<VEC> x[NV];
    float m = 0.f;
    FOR_PIECES(i, c) {
      load_piece<ODD, VEC, T>(xp, off, c, F, x[i]);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) m = max_abs(m, x[i].v[j]);
    }
    m = t.template reduce<false, true, false>(RowStats{0.f, 0.f, m}).mh;
    if (!t.ok) break;
    const float sc = row_scale(m);
    const RowInverse2 inv(row_inverse<sizeof(T) == 2>(sc, m));
    const uint32_t keep = not_finite(m) ? 0u : FULL;
    int8_t* qp = q + t.row * ld;
    FOR_PIECES(i, c) store_q<sizeof(T) == 2>(qp, c, x[i], inv, keep);
    for (long long c = (F + VEC - 1) / VEC * VEC + t.tid; c < ld; c += TEAM) qp[c] = 0;
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
    RowStats s{0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < F; c += blockDim.x) s.mh = max_abs(s.mh, load_one(xp + c), 0.f);
    s = block_reduce(s, red);
    const float sc = row_scale(s.mh);
    const RowInverse inv = row_inverse<sizeof(T) == 2>(sc, s.mh);
    const uint32_t keep = not_finite(s.mh) ? 0u : FULL;
    for (long long c = threadIdx.x; c < ld; c += blockDim.x) q[row * ld + c] = round1<sizeof(T) == 2>(c < F ? load_one(xp + c) : 0.f, inv, keep);
    if (threadIdx.x == 0) scale[row] = sc;
    __syncthreads();
  }
}

// ---------------------------------------------------------------- read back
// 16 values per thread; the caller made sure that the vectors of all rows can be counted in 32 bits.
template <class T>
__global__ void __launch_bounds__(256) dequantize_vec_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ y,
                                                             uint32_t vectors, uint32_t per_row, long long ld) {
  constexpr int VEC = 16 / sizeof(T), AT_ONCE = 2;
  for (uint32_t base = blockIdx.x * (256u * AT_ONCE) + threadIdx.x; base < vectors; base += gridDim.x * (256u * AT_ONCE)) {
    uint4 w[AT_ONCE];
    float s[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const uint32_t i = min(base + u * 256u, vectors - 1), row = i / per_row;
      w[u] = *reinterpret_cast<const uint4*>(q + row * ld + (i - row * per_row) * 16);
      s[u] = __ldg(scale + row);
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const uint32_t i = base + u * 256u;
      if (i >= vectors) break;
      const F2 s2(s[u], s[u]);
      F2 v[8];
      unpack4(w[u].x, v[0], v[1]); unpack4(w[u].y, v[2], v[3]); unpack4(w[u].z, v[4], v[5]); unpack4(w[u].w, v[6], v[7]);
      T* yp = y + static_cast<long long>(i) * 16;
#pragma unroll
      for (int k = 0; k < 16; k += VEC) {
        Piece<VEC> o;
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) o.v[j] = mul2(v[k / 2 + j], s2);
        store_vec(yp + k, o);
      }
    }
  }
}
// Row lengths that are no multiple of 16: the values in the order of memory, 8 to a thread from a 16-byte boundary on,
// whichever row they belong to. Their bytes are shifted out of the two aligned 8-byte words that hold them; pieces that
// reach into the next row go value by value. The caller made sure that the values can be counted in 32 bits.
template <class T>
__device__ __forceinline__ void store8(T* p, const F2* v) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = make_uint4(v[0].bf16(), v[1].bf16(), v[2].bf16(), v[3].bf16());
  } else {
    reinterpret_cast<ulonglong2*>(p)[0] = make_ulonglong2(v[0].v, v[1].v);
    reinterpret_cast<ulonglong2*>(p)[1] = make_ulonglong2(v[2].v, v[3].v);
  }
}
template <class T>
__global__ void __launch_bounds__(256) dequantize_odd_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ y,
                                                             uint32_t values, uint32_t F, long long ld) {
  constexpr int AT_ONCE = 4;
  const uint32_t pieces = (values + 7) / 8;
  for (uint32_t base = blockIdx.x * (256u * AT_ONCE) + threadIdx.x; base < pieces; base += gridDim.x * (256u * AT_ONCE)) {
    uint2 lo[AT_ONCE], hi[AT_ONCE];
    float s[AT_ONCE];
    uint32_t row[AT_ONCE], col[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const uint32_t i = min(base + u * 256u, pieces - 1);
      row[u] = i * 8 / F;
      col[u] = i * 8 - row[u] * F;
      const int8_t* p = q + row[u] * ld + (col[u] & ~7u);
      lo[u] = *reinterpret_cast<const uint2*>(p);
      hi[u] = (col[u] & 7) && col[u] + 8 <= F ? *reinterpret_cast<const uint2*>(p + 8) : make_uint2(0, 0);
      s[u] = __ldg(scale + row[u]);
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const uint32_t i = base + u * 256u;
      if (i >= pieces) break;
      T* yp = y + static_cast<long long>(i) * 8;
      if (col[u] + 8 <= F) {
        const bool words = col[u] & 4;
        const uint32_t bits = (col[u] & 3) * 8, a = words ? lo[u].y : lo[u].x, b = words ? hi[u].x : lo[u].y, c = words ? hi[u].y : hi[u].x;
        const F2 s2(s[u], s[u]);
        F2 v[4];
        unpack4(__funnelshift_r(a, b, bits), v[0], v[1]);
        unpack4(__funnelshift_r(b, c, bits), v[2], v[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], s2);
        store8(yp, v);
      } else {
        uint32_t r = row[u], c = col[u];
        for (uint32_t j = 0; j < min(8u, values - i * 8); ++j) {
          store_one(yp + j, static_cast<float>(q[r * ld + c]) * __ldg(scale + r));
          if (++c == F) {
            c = 0;
            ++r;
          }
        }
      }
    }
  }
}
// What that does not take: one warp per row.
template <class T>
__global__ void __launch_bounds__(256) dequantize_any_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ y,
                                                             long long rows, int F, long long ld) {
  const int lane = threadIdx.x & 31;
  for (long long row = blockIdx.x * 8ll + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8ll) {
    const float s = __ldg(scale + row);
#pragma unroll 8
    for (int c = lane; c < F; c += 32) {
      store_one(y + row * F + c, static_cast<float>(q[row * ld + c]) * s);
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
  float rstd, ymax, ys, hs;    // ymax: the largest |y|
  uint32_t keep_y, keep_h;     // all ones, or zero for a row that is not finite
  __device__ __forceinline__ void set_ymax(float m) {
    ymax = m;
    ys = row_scale(m);
    keep_y = not_finite(m) ? 0u : FULL;
  }
};
// h, its 8-bit rows and rstd follow from the sum of squares alone: a gamma that is not finite is y's affair.
__device__ __forceinline__ NormScales norm_scales(const RowStats& s, float inv_f, float eps) {
  NormScales r;
  const bool bad = not_finite(s.sq);           // a sum of squares: never negative; where it is finite, max |h| is
  const float var = s.sq * inv_f + eps;
  float t = rsqrtf(var);                       // within 2 ulp; one Newton step brings it to the rounding of 1 / sqrt
  t = fmaf(t, fmaf(var * t, -0.5f * t, 0.5f), t);   // var * t, a normal number, before the half: var need not be normal
  r.rstd = bad ? ROWS8_NAN : t;
  r.hs = bad ? ROWS8_NAN : row_scale(s.mh);
  r.keep_h = bad ? 0u : FULL;
  r.set_ymax(s.my * r.rstd);
  return r;
}
// rstd max |h gamma| stands for max |y|, but not where a product h gamma has left fp32's range and y = h rstd gamma need not
// have: above the range, or below its normal numbers with an rstd that brings it back (up to 1024, what is lost is less than
// 2^-13 of the smallest scale; with an eps of 1e-6 or more rstd is never larger, and a gamma of zeros costs nothing).
// Then the row's largest |y| is looked for once more, in the values that are quantised.
__device__ __forceinline__ bool ymax_is_lost(const RowStats& s, float rstd) {
  return s.mh > 0.f && !not_finite(s.sq) && (not_finite(s.my) || (s.my < ROWS8_TINY && rstd > 1024.f));
}
__device__ __forceinline__ void norm_row_done(const NormQ8Args& a, const NormScales& r, long long row) {
  a.ys[row] = r.ys;
  if (a.hq) a.hs[row] = r.hs;
  if (a.rstd) a.rstd[row] = r.rstd;
}

// One reduction serves both outputs: the largest |h gamma| times rstd is the largest |y| (but see ymax_is_lost), so sum h^2,
// max |h gamma| and max |h| are taken together and nothing waits for rstd. A row has been read whole before h is written (in
// place).
template <class T, int TEAM, bool ODD>
__global__ void __launch_bounds__(CTA, 1) rmsnorm_q8_kernel(const __grid_constant__ Ring ring, const NormQ8Args a) {
  constexpr int VEC = 16 / sizeof(T), NV = PER_THREAD / VEC, PAIRS = Piece<VEC>::PAIRS;
  extern __shared__ __align__(16) uint8_t smem[];
  Team<TEAM> t(ring, smem);
  t.template start<VEC>(a.gamma);
  const float* gamma = a.gamma ? reinterpret_cast<const float*>(smem + ring.gamma_at) : nullptr;
  const int F = ring.F;
  const float inv_f = 1.f / static_cast<float>(F);
  for (; t.row < ring.rows; t.template done<ODD && sizeof(T) == 4>()) {
    if (!t.template next<!(ODD && sizeof(T) == 4)>()) break;
    uint8_t* xp = t.bytes(0);
    const uint8_t* rp = ring.tensors > 1 ? t.bytes(1) : nullptr;
    const int off = ODD ? t.off(0) : 0;   // of x, residual and h alike
    T* hp = a.h ? static_cast<T*>(a.h) + t.row * F : nullptr;
    // x, residual and h have their own boundaries in common: h is written in their vectors, and where it is fp32 the sum
    // takes x's place in the ring, so that one tensor is left to be shifted.
    constexpr bool ADD_FIRST = ODD && sizeof(T) == 4;
    auto write_h = [&]() {
      const int end = off + F * static_cast<int>(sizeof(T));
      for (int at = t.tid * 16; at < end; at += TEAM * 16) {
        uint4 v = *reinterpret_cast<const uint4*>(xp + at);
        if (rp) v = add16<T>(v, *reinterpret_cast<const uint4*>(rp + at));
        if (ADD_FIRST && rp) *reinterpret_cast<uint4*>(xp + at) = v;
        if (hp) store_between(hp, off, at, F, v);
      }
    };
    if (ADD_FIRST) {
      write_h();
      t.sync();
    }
    Piece<VEC> h[NV];
    F2 sum[2] = {F2(0.f, 0.f), F2(0.f, 0.f)};
    RowStats s{0.f, 0.f, 0.f};
    FOR_PIECES(i, c) {
      load_piece<ODD, VEC, T>(xp, off, c, F, h[i]);
      if (!ADD_FIRST && rp) {
        Piece<VEC> r;
        load_piece<ODD, VEC, T>(rp, off, c, F, r);
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) h[i].v[j] = add2(h[i].v[j], r.v[j]);
      }
      Piece<VEC> gm;
      load_gamma(gamma, c, F, gm);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        F2& acc = sum[(i * PAIRS + j) & 1];
        acc = fma2(h[i].v[j], h[i].v[j], acc);
        s.my = max_abs(s.my, mul2(h[i].v[j], gm.v[j]));
        s.mh = max_abs(s.mh, h[i].v[j]);
      }
    }
    float even, odd;
    add2(sum[0], sum[1]).get(even, odd);
    s.sq = even + odd;
    s = t.template reduce<true, true, true>(s);
    if (!t.ok) break;
    NormScales r = norm_scales(s, inv_f, a.eps);
    const F2 rstd(r.rstd, r.rstd);
    if (ymax_is_lost(s, r.rstd)) {         // the same for all of the team
      float m = 0.f;
      FOR_PIECES(i, c) {
        Piece<VEC> gm;
        load_gamma(gamma, c, F, gm);
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) m = max_abs(m, mul2(mul2(h[i].v[j], rstd), gm.v[j]));
      }
      r.set_ymax(t.template reduce<false, false, true>(RowStats{0.f, m, 0.f}).my);
    }
    const RowInverse2 yi(row_inverse<true>(r.ys, r.ymax)), hi(row_inverse<false>(r.hs, s.mh));
    int8_t* yq = a.yq + t.row * a.ld;
    int8_t* hq = a.hq ? a.hq + t.row * a.ld : nullptr;
    FOR_PIECES(i, c) {
      if (!ODD && hp) store_vec(hp + c, h[i]);
      if (hq) store_q<false>(hq, c, h[i], hi, r.keep_h);
      Piece<VEC> y;
      load_gamma(gamma, c, F, y);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) y.v[j] = mul2(mul2(h[i].v[j], rstd), y.v[j]);
      store_q<true>(yq, c, y, yi, r.keep_y);
    }
    if (ODD && !ADD_FIRST && hp) write_h();
    for (long long c = (F + VEC - 1) / VEC * VEC + t.tid; c < a.ld; c += TEAM) {
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
    RowStats s{0.f, 0.f, 0.f};
    float h, gm;
    auto in = [&](long long c) {
      h = load_one(xp + c) + (rp ? load_one(rp + c) : 0.f);
      gm = a.gamma ? a.gamma[c] : 1.f;
    };
    for (int c = threadIdx.x; c < a.F; c += blockDim.x) {
      in(c);
      s.sq = fmaf(h, h, s.sq);
      s.my = max_abs(s.my, h * gm, 0.f);
      s.mh = max_abs(s.mh, h, 0.f);
    }
    s = block_reduce(s, red);
    NormScales n = norm_scales(s, 1.f / static_cast<float>(a.F), a.eps);
    if (ymax_is_lost(s, n.rstd)) {         // the same for the whole block
      RowStats y{0.f, 0.f, 0.f};
      for (int c = threadIdx.x; c < a.F; c += blockDim.x) {
        in(c);
        y.my = max_abs(y.my, h * n.rstd * gm, 0.f);
      }
      __syncthreads();                     // red has been read
      n.set_ymax(block_reduce(y, red).my);
    }
    const RowInverse yi = row_inverse<true>(n.ys, n.ymax), hi = row_inverse<false>(n.hs, s.mh);
    for (long long c = threadIdx.x; c < a.ld; c += blockDim.x) {
      h = gm = 0.f;
      if (c < a.F) {
        in(c);
        if (a.h) store_one(static_cast<T*>(a.h) + row * a.F + c, h);
      }
      if (a.hq) a.hq[row * a.ld + c] = round1<false>(h, hi, n.keep_h);
      a.yq[row * a.ld + c] = round1<true>(h * n.rstd * gm, yi, n.keep_y);
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
template <class T, int TEAM, bool ODD>
__global__ void __launch_bounds__(CTA, 1) rmsnorm_bwd_kernel(const __grid_constant__ Ring ring, const NormBwdQ8Args a) {
  constexpr int VEC = 16 / sizeof(T), NV = PER_THREAD / VEC, PAIRS = Piece<VEC>::PAIRS;
  constexpr bool ADD_LAST = ODD && sizeof(T) == 4;   // rstd and the residual's gradient come in as the row leaves the ring
  extern __shared__ __align__(16) uint8_t smem[];
  Team<TEAM> t(ring, smem);
  t.template start<VEC>(a.gamma);
  const float* gamma = a.gamma ? reinterpret_cast<const float*>(smem + ring.gamma_at) : nullptr;
  const int F = ring.F;
  const float inv_f = 1.f / static_cast<float>(F);
  Piece<VEC> acc[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) acc[i].v[j] = F2(0.f, 0.f);
  float row_rstd = 0.f, row_scale8 = 0.f;   // of the next row: they come from memory while this one is worked on
  if (t.row < ring.rows) {
    row_rstd = __ldg(a.rstd + t.row);
    row_scale8 = __ldg(a.hs + t.row);
  }
  for (; t.row < ring.rows; t.template done<ODD>()) {
    const float rstd = row_rstd, s = row_scale8 * rstd;
    const F2 s2(s, s), rstd2(rstd, rstd);
    t.template next<true>();
    if (t.row + t.step < ring.rows) {
      row_rstd = __ldg(a.rstd + t.row + t.step);
      row_scale8 = __ldg(a.hs + t.row + t.step);
    }
    const uint8_t* qp = t.bytes(0);
    uint8_t* gp = t.bytes(1);
    const uint8_t* rp = ring.tensors > 2 ? t.bytes(2) : nullptr;
    const int off = ODD ? t.off(1) : 0;
    F2 dots[2] = {F2(0.f, 0.f), F2(0.f, 0.f)};
    FOR_PIECES(i, c) {
      Piece<VEC> g, n, gm;
      load_piece<ODD, VEC, T>(gp, off, c, F, g);
      load_q(qp, c, n);
      load_gamma(gamma, c, F, gm);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        n.v[j] = mul2(n.v[j], s2);
        acc[i].v[j] = fma2(g.v[j], n.v[j], acc[i].v[j]);
        F2& dot = dots[(i * PAIRS + j) & 1];
        dot = fma2(mul2(g.v[j], gm.v[j]), n.v[j], dot);
      }
    }
    float even, odd;
    add2(dots[0], dots[1]).get(even, odd);
    const float dot = t.template reduce<true, false, false>(RowStats{even + odd, 0.f, 0.f}).sq * inv_f;
    if (!t.ok) break;
    const F2 back(-s * dot, -s * dot);       // the row's part along n, for the bytes of n
    T* op = static_cast<T*>(a.gh) + t.row * F;
    FOR_PIECES(i, c) {
      Piece<VEC> g, n, r;
      load_piece<ODD, VEC, T>(gp, off, c, F, g);
      load_q(qp, c, n);
      load_gamma(gamma, c, F, r);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) g.v[j] = fma2(n.v[j], back, mul2(g.v[j], r.v[j]));
      if (ADD_LAST) {
      } else if (rp) {
        load_piece<ODD, VEC, T>(rp, off, c, F, r);
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) g.v[j] = fma2(g.v[j], rstd2, r.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) g.v[j] = mul2(g.v[j], rstd2);
      }
      if (ODD) place_piece(gp, off, c, g);   // its own bytes of grad_out, which nobody reads again
      else store_vec(op + c, g);
    }
    if (ODD) {         // then out of the ring in the vectors that memory has
      t.sync();
      const int end = off + F * static_cast<int>(sizeof(T));
      for (int at = t.tid * 16; at < end; at += TEAM * 16) {
        uint4 v = *reinterpret_cast<const uint4*>(gp + at);
        if constexpr (ADD_LAST) {
          Piece<VEC> g, r;
          load_vec(reinterpret_cast<const float*>(gp + at), g);
          r.v[0] = r.v[1] = F2(-0.f, -0.f);
          if (rp) load_vec(reinterpret_cast<const float*>(rp + at), r);
#pragma unroll
          for (int j = 0; j < PAIRS; ++j) g.v[j] = fma2(g.v[j], rstd2, r.v[j]);
          v = make_uint4(static_cast<uint32_t>(g.v[0].v), static_cast<uint32_t>(g.v[0].v >> 32), static_cast<uint32_t>(g.v[1].v), static_cast<uint32_t>(g.v[1].v >> 32));
        }
        store_between(op, off, at, F, v);
      }
    }
  }
  t.end();
  if (!a.partial) return;
  // the teams' sums side by side in the ring's memory (teams * F <= 512 * 32: every row that was fetched has been waited
  // for), then added in the teams' order
  float* columns = reinterpret_cast<float*>(smem + ring.slots_at);
  float* mine = columns + t.team * F;
  FOR_PIECES(i, c) {
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      float lo, hi;
      acc[i].v[j].get(lo, hi);
      if (!ODD || c + 2 * j < F) mine[c + 2 * j] = lo;
      if (!ODD || c + 2 * j + 1 < F) mine[c + 2 * j + 1] = hi;
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < F; c += CTA) {
    float sum = columns[c];
#pragma unroll
    for (int w = 1; w < CTA / TEAM; ++w) sum += columns[w * F + c];
    a.partial[static_cast<long long>(blockIdx.x) * F + c] = sum;
  }
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
    RowStats st{0.f, 0.f, 0.f};
    auto scaled = [&](int c) { return load_one(gp + c) * (a.gamma ? a.gamma[c] : 1.f); };
    for (int c = threadIdx.x; c < a.F; c += blockDim.x) st.sq = fmaf(scaled(c), static_cast<float>(qp[c]) * s, st.sq);
    const float dot = block_reduce(st, red).sq / static_cast<float>(a.F);
    for (int c = threadIdx.x; c < a.F; c += blockDim.x)
      store_one(op + c, rstd * (scaled(c) - static_cast<float>(qp[c]) * s * dot) + (rp ? load_one(rp + c) : 0.f));
    __syncthreads();
  }
}
template <class T>
__global__ void __launch_bounds__(256) rmsnorm_bwd_long_columns_kernel(const NormBwdQ8Args a, long long rows_per_block) {
  const long long r0 = static_cast<long long>(blockIdx.x) * rows_per_block;
  const long long r1 = min(a.rows, r0 + rows_per_block);
  for (int f = threadIdx.x; f < a.F; f += blockDim.x) {
    float acc = 0.f;
    for (long long r = r0; r < r1; ++r)
      acc = fmaf(load_one(static_cast<const T*>(a.go) + r * a.F + f), static_cast<float>(a.hq[r * a.ld + f]) * (a.hs[r] * a.rstd[r]), acc);
    a.partial[static_cast<long long>(blockIdx.x) * a.F + f] = acc;
  }
}
__global__ void __launch_bounds__(512) sum_partials_kernel(const float* partial, float* out, int blocks, int F) {
  __shared__ float part[16][33];
  wait_for_previous_kernel();
  column_total(partial, out, blocks, F, static_cast<int>(blockIdx.x), part);
}

// ---------------------------------------------------------------- launch shapes
bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  return true;
}
constexpr int RING_BYTES = 216 * 1024;

// The ring's geometry, for rows of up to 512 * 32 values that fit shared memory, on tensors that start on
// 16-byte boundaries. It depends on the row's length alone, so a row's sums have the same order, and its
// result the same bits, in every batch.
struct RowTensor {
  const void* p;
  long long pitch, bytes;   // from row to row, and of a row (more than an int holds where the ring does not take them)
};
// Returns the threads per row, or 0.
int make_ring(grilly_ctx* ctx, Ring& g, long long rows, int F, const RowTensor* tensors, int count, bool gamma, bool gamma_sums, size_t* smem, unsigned* grid) {
  if (F > CTA * PER_THREAD) return 0;
  g = Ring{};
  g.rows = rows;
  g.F = F;
  g.err = ctx->err_dev;
  g.tensors = count;
  g.aligned = 1;
  g.first_tail = rows;
  for (int i = 0; i < count; ++i) {
    if (reinterpret_cast<uintptr_t>(tensors[i].p) & 15) return 0;
    g.src[i] = tensors[i].p;
    g.pitch[i] = tensors[i].pitch;
    g.bytes[i] = static_cast<int>(tensors[i].bytes);
    g.total[i] = tensors[i].pitch * (rows - 1) + tensors[i].bytes;
    const long long whole = g.total[i] & ~15ll;
    g.first_tail = std::min(g.first_tail, whole < g.bytes[i] ? 0 : (whole - g.bytes[i]) / g.pitch[i] + 1);
    g.at[i] = g.slot;
    if (g.pitch[i] % 16 || g.bytes[i] % 16) g.aligned = 0;
    g.slot += (g.bytes[i] + 15) / 16 * 16 + (tensors[i].pitch % 16 ? 16 : 0);
  }
  g.gamma_at = GAMMA_AT;
  g.slots_at = GAMMA_AT + (gamma ? (F + 7) / 8 * 32 : 0);
  // the smallest team that holds a row, but few enough of them that each has two rows in shared memory: the threads that
  // long rows leave without a row of their own join the others. Rows of which only one fits are loaded one after the other
  // (5000 x 11001 fp32: the norm 196 us, its backward pass 200; read twice from memory instead 413 and 838)
  const int room = RING_BYTES - g.slots_at;
  int team = MIN_TEAM;
  while (team < CTA && (team * PER_THREAD < F || CTA / team * 2 * g.slot > room)) team *= 2;
  const int teams = CTA / team;
  if (teams * g.slot > room) return 0;
  *grid = static_cast<unsigned>(std::min<long long>(rows, ctx->num_sms));
  const long long per_team = (rows + static_cast<long long>(*grid) * teams - 1) / (static_cast<long long>(*grid) * teams);
  g.depth = static_cast<int>(std::min<long long>(std::min(MAX_DEPTH, room / (g.slot * teams)), per_team));
  *smem = g.slots_at + std::max(static_cast<size_t>(g.slot) * teams * g.depth, gamma_sums ? sizeof(float) * static_cast<size_t>(F) * teams : 0);
  return team;
}
// CALL(TEAM) for the team of a ring
#define WITH_TEAM(team, CALL)      \
  switch (team) {                  \
    case 16: CALL(16); break;      \
    case 32: CALL(32); break;      \
    case 64: CALL(64); break;      \
    case 128: CALL(128); break;    \
    case 256: CALL(256); break;    \
    default: CALL(512);            \
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
  Ring ring;
  size_t smem;
  unsigned grid;
  const long long pitch = static_cast<long long>(sizeof(T)) * F;
  const RowTensor in[1] = {{x, pitch, pitch}};
  const int team = make_ring(ctx, ring, rows, F, in, 1, false, false, &smem, &grid);
  if (!team) {
    quantize_long_rows_kernel<<<any_grid(rows), 1024, 0, ctx->stream>>>(x, q, scale, rows, F, ld);
    return GRILLY_OK;
  }
  void (*kern)(const Ring, int8_t*, float*, long long) = nullptr;
#define PICK(TEAM) kern = ring.aligned ? quantize_rows_kernel<T, TEAM, false> : quantize_rows_kernel<T, TEAM, true>
  WITH_TEAM(team, PICK)
#undef PICK
  if (int rc = allow_ring(ctx, kern)) return rc;
  kern<<<grid, CTA, smem, ctx->stream>>>(ring, q, scale, ld);
  return GRILLY_OK;
}

template <class T>
void launch_dequantize(grilly_ctx* ctx, const int8_t* q, const float* scale, T* y, long long rows, int F, long long ld) {
  const cudaStream_t st = ctx->stream;
  const long long vectors = rows * (F / 16);
  if (F % 16 == 0 && aligned16({y}) && vectors < (1ll << 31)) {
    const unsigned grid = static_cast<unsigned>(std::min<long long>((vectors + 511) / 512, ctx->num_sms * 32ll));
    dequantize_vec_kernel<T><<<grid, 256, 0, st>>>(q, scale, y, static_cast<uint32_t>(vectors), static_cast<uint32_t>(F / 16), ld);
  } else if (aligned16({y}) && rows * F < (1ll << 32) - 4096 && rows * F > 0) {
    const long long pieces = (rows * F + 7) / 8;
    const unsigned grid = static_cast<unsigned>(std::min<long long>((pieces + 1023) / 1024, ctx->num_sms * 16ll));
    dequantize_odd_kernel<T><<<grid, 256, 0, st>>>(q, scale, y, static_cast<uint32_t>(rows * F), static_cast<uint32_t>(F), ld);
  } else {
    dequantize_any_kernel<T><<<any_grid((rows + 7) / 8), 256, 0, st>>>(q, scale, y, rows, F, ld);
  }
}

template <class T>
int launch_rmsnorm(grilly_ctx* ctx, const NormQ8Args& a) {
  Ring ring;
  size_t smem;
  unsigned grid;
  const long long pitch = static_cast<long long>(sizeof(T)) * a.F;
  const RowTensor in[2] = {{a.x, pitch, pitch}, {a.residual, pitch, pitch}};
  const int team = aligned16({a.h}) ? make_ring(ctx, ring, a.rows, a.F, in, a.residual ? 2 : 1, a.gamma != nullptr, false, &smem, &grid) : 0;
  if (!team) {
    rmsnorm_q8_long_kernel<T><<<any_grid(a.rows), 1024, 0, ctx->stream>>>(a);
    return GRILLY_OK;
  }
  void (*kern)(const Ring, const NormQ8Args) = nullptr;
#define PICK(TEAM) kern = ring.aligned ? rmsnorm_q8_kernel<T, TEAM, false> : rmsnorm_q8_kernel<T, TEAM, true>
  WITH_TEAM(team, PICK)
#undef PICK
  if (int rc = allow_ring(ctx, kern)) return rc;
  kern<<<grid, CTA, smem, ctx->stream>>>(ring, a);
  return GRILLY_OK;
}

template <class T>
int launch_rmsnorm_bwd(grilly_ctx* ctx, NormBwdQ8Args& a, float* grad_gamma) {
  Rows8Scratch scratch(ctx);
  Ring ring;
  size_t smem;
  unsigned grid;
  const long long pitch = static_cast<long long>(sizeof(T)) * a.F;
  const RowTensor in[3] = {{a.hq, a.ld, (a.F + 15) / 16 * 16}, {a.go, pitch, pitch}, {a.gr, pitch, pitch}};
  const int team = aligned16({a.gh}) ? make_ring(ctx, ring, a.rows, a.F, in, a.gr ? 3 : 2, a.gamma != nullptr, grad_gamma != nullptr, &smem, &grid) : 0;
  if (team) {
    void (*kern)(const Ring, const NormBwdQ8Args) = nullptr;
#define PICK(TEAM) kern = ring.aligned ? rmsnorm_bwd_kernel<T, TEAM, false> : rmsnorm_bwd_kernel<T, TEAM, true>
    WITH_TEAM(team, PICK)
#undef PICK
    if (int rc = allow_ring(ctx, kern)) return rc;
    if (grad_gamma) {
      const size_t at = scratch.reserve(sizeof(float) * grid * static_cast<size_t>(a.F));
      if (int rc = scratch.take()) return rc;
      a.partial = scratch.at<float>(at);
    }
    kern<<<grid, CTA, smem, ctx->stream>>>(ring, a);
    ctx->launches++;
    if (grad_gamma) {
      GB_CUDA_CHECK(ctx, launch_following(ctx->stream, sum_partials_kernel, (a.F + 31) / 32, 512, a.partial, grad_gamma, static_cast<int>(grid), a.F));
      ctx->launches++;
    }
    GB_CUDA_CHECK(ctx, cudaGetLastError());
    return GRILLY_OK;
  }
  if (grad_gamma) {
    const int blocks = static_cast<int>(std::min<long long>((a.rows + 31) / 32, ctx->num_sms));
    const long long per = (a.rows + blocks - 1) / blocks;
    const size_t at = scratch.reserve(sizeof(float) * blocks * static_cast<size_t>(a.F));
    if (int rc = scratch.take()) return rc;
    a.partial = scratch.at<float>(at);
    rmsnorm_bwd_long_columns_kernel<T><<<blocks, 256, 0, ctx->stream>>>(a, per);
    GB_CUDA_CHECK(ctx, launch_following(ctx->stream, sum_partials_kernel, (a.F + 31) / 32, 512, a.partial, grad_gamma, blocks, a.F));
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
    const int elt = bf16 ? 2 : 4;
    const Rows8Span outs[] = {{q, rows * ld}, {scale, 4 * rows}}, ins[] = {{x, rows * features * elt, 0, elt}};
    if (int rc = rows8_memory(ctx, "quantize_rows", outs, ins)) return rc;
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
    const int elt = bf16 ? 2 : 4;
    const Rows8Span outs[] = {{y, rows * features * elt, 0, elt}}, ins[] = {{q, rows * ld}, {scale, 4 * rows}};
    if (int rc = rows8_memory(ctx, "dequantize_rows", outs, ins)) return rc;
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
    const int elt = bf16 ? 2 : 4;
    const long long size = rows * features * elt;
    const Rows8Span outs[] = {{h, size, 0, elt}, {y_q, rows * ld}, {y_scale, 4 * rows}, {h_q, rows * ld}, {h_scale, 4 * rows}, {rstd, 4 * rows}};
    const Rows8Span ins[] = {{x, size, 1, elt}, {residual, size, 1, elt}, {gamma, 4ll * features}};
    if (int rc = rows8_memory(ctx, "rmsnorm_residual_q8", outs, ins)) return rc;
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
    const int elt = bf16 ? 2 : 4;
    const long long size = rows * features * elt;
    const Rows8Span outs[] = {{grad_h, size, 0, elt}, {grad_gamma, 4ll * features}};
    const Rows8Span ins[] = {{go, size, 1, elt}, {grad_residual, size, 1, elt}, {h_q, rows * ld}, {h_scale, 4 * rows}, {rstd, 4 * rows}, {gamma, 4ll * features}};
    if (int rc = rows8_memory(ctx, "rmsnorm_backward_q8", outs, ins)) return rc;
    NormBwdQ8Args a{go, static_cast<const int8_t*>(h_q), h_scale, rstd, gamma, grad_residual, grad_h, nullptr, rows, ld, features};
    const double e = bf16 ? 2 : 4, n = static_cast<double>(rows) * features;
    const int pi = prof_begin(ctx, PROF_NORM, 10.0 * n, n * (e * (2 + (grad_residual ? 1 : 0)) + 1) + 8.0 * features + 8.0 * rows);
    const int rc = bf16 ? launch_rmsnorm_bwd<__nv_bfloat16>(ctx, a, grad_gamma) : launch_rmsnorm_bwd<float>(ctx, a, grad_gamma);
    prof_end(ctx, pi);
    return rc;
  });
}

}  // extern "C"
