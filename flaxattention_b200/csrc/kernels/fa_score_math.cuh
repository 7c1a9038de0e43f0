// Quotients and tanh of scores, for score_mods of 16-bit inputs (capped scores), without branches: with them, the scores of a thread are computed
// one behind the other (20 rows over 18944 tiles of 32 keys, D 128: 120 us with tanhf, 71 without a mod).  The lowering writes FA_QUOTIENT, FA_QUOTIENT_BY
// (a constant) and FA_TANH only where the value depends on the score and stays one: what reaches a comparison, a rounding, a whole number or a
// table, and all that does not read the score, is divided exactly, as every mask is.
//
// Quotients are off by two units in the last place of fp32 at most (a score of 30 by 4e-6, its probability by as much in proportion, where the
// rounding of results to fp16 takes 5e-4).  tanh: where the value is small, its Taylor series up to x^13, whose next term is below 2^-24 of it;
// else 1 - 2 / (exp(2 x) + 1), off by some 2^-22.  Both are worked out and one is taken.
#pragma once
__device__ __forceinline__ float fa_quotient(float a, float b) {
  float r;
  asm("div.full.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
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
#define FA_QUOTIENT(a, b) fa_quotient(a, b)
#define FA_QUOTIENT_BY(a, c) ((a) * (1.0f / (c)))
#define FA_TANH(x) fa_tanh(x)
