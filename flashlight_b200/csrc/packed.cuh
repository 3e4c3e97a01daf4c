// Pairs of fp32 numbers in one register pair: an instruction works on both, each rounded as it would be alone.
#pragma once
#include <cuda_runtime.h>

namespace flb200 {

struct F2 {
  unsigned long long r;
};
__device__ __forceinline__ F2 pair(float a, float b) {
  F2 x;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x.r) : "f"(a), "f"(b));
  return x;
}
__device__ __forceinline__ F2 pair(float a) { return pair(a, a); }
__device__ __forceinline__ void unpair(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.r));
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 x;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x.r) : "l"(a.r), "l"(b.r));
  return x;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 x;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(x.r) : "l"(a.r), "l"(b.r));
  return x;
}
__device__ __forceinline__ F2 fused(F2 a, F2 b, F2 c) {  // a b + c
  F2 x;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x.r) : "l"(a.r), "l"(b.r), "l"(c.r));
  return x;
}
}  // namespace flb200
