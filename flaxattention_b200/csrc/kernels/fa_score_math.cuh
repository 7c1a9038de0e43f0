// Quotients and tanh of scores, for score_mods of 16-bit inputs (capped scores), without branches: with them, the scores of a thread are computed
// one behind the other (20 rows over 18944 tiles of 32 keys, D 128: 120 us with tanhf, 71 without a mod).  The lowering writes FA_QUOTIENT, FA_QUOTIENT_BY
// (a constant) and FA_TANH only where the value depends on the score and stays one: what reaches a comparison, a rounding, a whole number or a
// table, and all that does not read the score, is divided exactly, as every mask is.
//
// Quotients are off by two units in the last place of fp32 at most (a score of 30 by 4e-6, its probability by as much in proportion, where the
// rounding of results to fp16 takes 5e-4).  tanh: where the value is small, its Taylor series up to x^13, whose next term is below 2^-24 of it;
// else 1 - 2 / (exp(2 x) + 1), off by some 2^-22.  Both are worked out and one is taken.
//
// Kernels that define FA_PAIRS (of prompts, over a shared prefix, over 8-bit pages; over pages of 16 bits results stay as they were) have another:
// x P(x^2) / Q(x^2), P and Q of degree 4, on [-8.3, 8.3], beyond which tanh is 1 to fp32.  The coefficients are the least largest relative error's
// (9.4e-9; least squares, reweighted until the errors were level), all of one sign, so that nothing cancels: off by 4e-7 in proportion with the
// roundings and the reciprocal's, the same for small values as for large.  One SFU operation instead of two, and of two scores at once half the
// instructions (FA_SCORE_PAIRS: the lowering's form of a score_mod for two keys): 9 a score instead of 17.  (5 prompts' pieces of up to 777 behind up
// to 3001, 12 / 4 heads, D 80, fp16: 168 us, so 125.)
#pragma once
#if FA_PAIRS
#include "fa_f2.cuh"  // (and nothing that has fa_params.h in it: this stands in front of the mods, and that asks whether they read tensors)
#endif
__device__ __forceinline__ float fa_quotient(float a, float b) {
  float r;
  asm("div.full.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
#if FA_PAIRS
__device__ __forceinline__ float fa_tanh_range(float x) {  // (no number stays none)
  float r;
  asm("min.NaN.f32 %0, %1, 0f4104CCCD;\n\tmax.NaN.f32 %0, %0, 0fC104CCCD;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fa_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ fa_u64 fa_both(float x) { return fa_f2(x, x); }
__device__ __forceinline__ fa_u64 fa_tanh2(fa_u64 x) {
  float a, b;
  fa_f2_unpack(x, a, b);
  x = fa_f2(fa_tanh_range(a), fa_tanh_range(b));
  const fa_u64 s = fa_mul2(x, x);
  fa_u64 p = fa_fma2(s, fa_both(1.464823906616175e-08f), fa_both(2.1508480131160468e-05f));
  p = fa_fma2(p, s, fa_both(0.0035491681192070246f));
  p = fa_fma2(p, s, fa_both(0.1342587023973465f));
  p = fa_fma2(p, s, fa_both(1.f));
  fa_u64 q = fa_fma2(s, fa_both(8.295099860333721e-07f), fa_both(0.0003373948857188225f));
  q = fa_fma2(q, s, fa_both(0.026079945266246796f));
  q = fa_fma2(q, s, fa_both(0.46759194135665894f));
  q = fa_fma2(q, s, fa_both(1.f));
  fa_f2_unpack(q, a, b);
  return fa_mul2(fa_mul2(x, p), fa_f2(fa_rcp(a), fa_rcp(b)));
}
__device__ __forceinline__ float fa_tanh(float x) {
  x = fa_tanh_range(x);
  const float s = x * x;
  float p = fmaf(s, 1.464823906616175e-08f, 2.1508480131160468e-05f);
  p = fmaf(p, s, 0.0035491681192070246f);
  p = fmaf(p, s, 0.1342587023973465f);
  p = fmaf(p, s, 1.f);
  float q = fmaf(s, 8.295099860333721e-07f, 0.0003373948857188225f);
  q = fmaf(q, s, 0.026079945266246796f);
  q = fmaf(q, s, 0.46759194135665894f);
  q = fmaf(q, s, 1.f);
  return x * p * fa_rcp(q);
}
#else
__device__ __forceinline__ float fa_tanh(float x) {
  const float s = x * x;
  float t = 21844.f / 6081075.f;
  t = fmaf(t, s, -1382.f / 155925.f);
  t = fmaf(t, s, 62.f / 2835.f);
  t = fmaf(t, s, -17.f / 315.f);
  t = fmaf(t, s, 2.f / 15.f);
  t = fmaf(t, s, -1.f / 3.f);
  t = fmaf(t * s, x, x);
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 2.8853900817779268f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.f));
  const float far = fmaf(-2.f, r, 1.f);
  return s < 0.16f ? t : far;  // (no number: neither is)
}
#endif
#define FA_QUOTIENT(a, b) fa_quotient(a, b)
#define FA_QUOTIENT_BY(a, c) ((a) * (1.0f / (c)))
#define FA_TANH(x) fa_tanh(x)
