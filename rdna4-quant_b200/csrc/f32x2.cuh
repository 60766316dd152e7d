// Pairs of floats in one 64-bit register: an instruction of the fp32 pipe does two
// operations (add, mul and fma with f32x2 operands, each rounded as the scalar one).
#pragma once
#include <stdint.h>

namespace r4q {

struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit F2(uint64_t u) : v(u) {}
  __device__ __forceinline__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
__device__ __forceinline__ F2 add(F2 a, F2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v));
  return F2(d);
}
__device__ __forceinline__ F2 sub(F2 a, F2 b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v));
  return F2(d);
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v));
  return F2(d);
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a.v), "l"(b.v), "l"(c.v));
  return F2(d);
}

}  // namespace r4q
