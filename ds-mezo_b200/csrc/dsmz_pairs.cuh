// Two fp32 in one register pair: the packed add, multiply and multiply-add take one issue slot
// for both.
#pragma once

#include <stdint.h>

namespace dsmz {

struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ explicit F2(float a) { asm("mov.b64 %0, {%1, %1};" : "=l"(v) : "f"(a)); }
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void split(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 c;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}
__device__ __forceinline__ F2 add_down(F2 a, F2 b) {        // rounded towards minus infinity
  F2 c;
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 c;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}

}  // namespace dsmz
