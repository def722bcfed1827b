// Softmax statistics that the scoring kernels share.  A tally of some scores x under the factor c = log2(e) / temperature:
//
//   m = max x        z = sum 2^t        s = sum 2^t t        with t = (x - m) c
//
// so that of a whole row   log softmax(x[i]) = (x[i] - m) / temperature - log z   and the entropy in bits is   log2 z - s / z.
// Everything is relative to m, where fp32 loses nothing: the sums of terms relative to 0 would cancel.
// -inf adds nothing; NaN and +inf make z NaN, and with it every result of the row.  The tally of nothing is {-FLT_MAX, 0, 0}.
#pragma once
#include <cfloat>

#include "common.cuh"

namespace xllm {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Tally {
  float m, z, s;
};

__device__ __forceinline__ float exp2_fast(float t) {          // 2^-22 relative, 0 below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// t from below so that 0 * -inf does not meet in s; NaN stays NaN
__device__ __forceinline__ float bounded(float t) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(t), "f"(-1024.f));
  return r;
}
__device__ __forceinline__ Tally tally_empty() { return {-FLT_MAX, 0.f, 0.f}; }
// the same tally relative to a maximum m >= a.m
__device__ __forceinline__ void tally_rebase(Tally& a, float m, float c) {
  const float d = bounded((a.m - m) * c), f = exp2_fast(d);
  a.s = f * fmaf(d, a.z, a.s);
  a.z *= f;
  a.m = m;
}
__device__ __forceinline__ Tally tally_join(Tally a, Tally b, float c) {
  const float m = fmaxf(a.m, b.m);
  tally_rebase(a, m, c);
  tally_rebase(b, m, c);
  return {m, a.z + b.z, a.s + b.s};
}
// Pairs of fp32 in one instruction.
typedef float2 f32x2;
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { return __ffma2_rn(a, b, c); }

// A tally that takes two scores at a time: its sums are those of the first and of the second ones.
struct PairTally {
  float m;
  f32x2 z, s;
};
__device__ __forceinline__ PairTally pair_empty() { return {-FLT_MAX, {0.f, 0.f}, {0.f, 0.f}}; }
__device__ __forceinline__ void pair_rebase(PairTally& a, float m, float c) {      // m >= a.m
  const float d = bounded((a.m - m) * c), f = exp2_fast(d);
  a.s = mul2({f, f}, fma2({d, d}, a.z, a.s));
  a.z = mul2({f, f}, a.z);
  a.m = m;
}
__device__ __forceinline__ void pair_add(PairTally& a, f32x2 x, float c) {         // neither is above a.m
  f32x2 t = mul2(add2(x, {-a.m, -a.m}), {c, c});
  t = {bounded(t.x), bounded(t.y)};
  const f32x2 e = {exp2_fast(t.x), exp2_fast(t.y)};
  a.z = add2(a.z, e);
  a.s = fma2(e, t, a.s);
}
__device__ __forceinline__ Tally pair_sum(const PairTally& a) { return {a.m, a.z.x + a.z.y, a.s.x + a.s.y}; }

// 1 / temperature of a row; c is log2(e) times it.  Both are finite: below 2.9e-39 the inverse would not be, and what is 0 behind the
// maximum would be NaN; a temperature that low leaves the same tokens as 5e-39.
__device__ __forceinline__ float row_scale(const float* temperature, int64_t row) {
  const float t = temperature ? temperature[row] : 1.f;
  return t > 0.f ? 1.f / fmaxf(t, 5e-39f) : 1.f;
}
// in nats: the type's lowest value as a score leaves fp32's range when scaled to bits
__device__ __forceinline__ float tally_logprob(const Tally& a, float x, float scale) {
  return a.z == 0.f ? -INFINITY : (x - a.m) * scale - logf(a.z);
}
__device__ __forceinline__ float tally_entropy(const Tally& a) {
  return a.z == 0.f ? 0.f : (log2f(a.z) - a.s / a.z) * kLn2;
}

}  // namespace xllm
