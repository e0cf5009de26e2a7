// Two fp32 values in one 64-bit register pair: one instruction for two products or sums (sm_100).
#pragma once
#include <cstdint>
#include <cuda_bf16.h>

namespace gb {

struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
  __device__ __forceinline__ uint32_t bf16() const {   // both rounded to bf16, packed
    float a, b;
    get(a, b);
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return d; }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { F2 d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
__device__ __forceinline__ F2 add2(F2 a, F2 b) { F2 d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
// the largest of m, |a|, |b|; a NaN wins
__device__ __forceinline__ float max_abs(float m, float a, float b) {
  asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float max_abs(float m, F2 x) {
  float a, b;
  x.get(a, b);
  return max_abs(m, a, b);
}

}  // namespace gb
