// Two fp32 values in a 64-bit register, computed with at once (sm_100).  Includes nothing: fa_score_math.cuh, which stands in front of the mods, has it too.
#pragma once
typedef unsigned long long fa_u64;

__device__ __forceinline__ fa_u64 fa_f2(float lo, float hi) {
  fa_u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void fa_f2_unpack(fa_u64 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ fa_u64 fa_mul2(fa_u64 a, fa_u64 b) {
  fa_u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ fa_u64 fa_add2(fa_u64 a, fa_u64 b) {
  fa_u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ fa_u64 fa_fma2(fa_u64 a, fa_u64 b, fa_u64 c) {
  fa_u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
