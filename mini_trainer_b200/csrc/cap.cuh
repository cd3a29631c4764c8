// Numbers capped by a tanh, unit tanh(scale s / cap): attention wants them in units of log2 e, as its exponentials do (unit = cap log2 e), the head as a part of the cap (1).
//
// Up to the cap (|scale s| <= cap) an odd polynomial of degree eleven on [-1, 1], 6.8e-7 off at most, with the powers of scale / cap in its coefficients: seven packed
// instructions for two numbers; up to half of it one of degree seven on [-1/2, 1/2] (5.7e-7), five. Beyond the cap tanh as 1 - 2 / (1 + e^2x), two operations on the special-function
// unit each, whose error is 2^-22 of the cap: a softmax that is bound by that unit as it is would do three times the work there. A tile in which one score is beyond the cap takes that form
// throughout, so batches whose scores fill the cap take it nearly everywhere (attention_rule.cuh has the times).
#pragma once
#include <stdint.h>

#include "ptx.cuh"

namespace mtb {

// The polynomial: tanh(x) = x (C0 + C1 x^2 + ...).
constexpr float CAP_C[6] = {0.99999949f, -0.33329398f, 0.13284259f, -0.05168433f, 0.01683263f, -0.00310275f};
constexpr float CAP_HALF[4] = {0.99999948f, -0.33326467f, 0.13191882f, -0.04444443f};

struct CapArgs {
  float2 a[6];       // twice each, for packed arithmetic: s (a0 + a1 s^2 + ...)
  float2 b[4];       // the same of degree seven
  float most, low;   // |s| up to which they hold; `low` also keeps capped numbers within +-30
  float unit, k2;    // k2: 2 scale / cap log2 e
  float inv2;        // -1 / unit^2: the derivative is 1 + inv2 v^2 of a capped number v
};

// Range of caps. Above it the exact form's error would pass 1e-3 of the scale's unit.
inline bool cap_ok(float scale, float cap) { return scale > 0.f && cap > 0.f && scale >= cap * 0x1p-13f && scale <= cap * 0x1p10f; }

inline CapArgs cap_args(float scale, float cap, double unit) {
  CapArgs r{};
  const double k = static_cast<double>(scale) / cap;
  double p = k;
  for (int i = 0; i < 4; ++i, p *= k * k) r.b[i].x = r.b[i].y = static_cast<float>(unit * CAP_HALF[i] * p);
  p = k;
  for (int i = 0; i < 6; ++i, p *= k * k) r.a[i].x = r.a[i].y = static_cast<float>(unit * CAP_C[i] * p);
  r.most = k >= 0x1p-11 ? static_cast<float>(1.0 / k) : -1.f;   // below, k^11 is no normal number: the exact form throughout
  r.low = r.most * static_cast<float>(unit > 60.0 ? 30.0 / unit : 0.5);
  r.unit = static_cast<float>(unit);
  r.k2 = static_cast<float>(2.0 * k * 1.4426950408889634);
  r.inv2 = static_cast<float>(-1.0 / (unit * unit));
  return r;
}

// Any argument: infinities saturate.
__device__ __forceinline__ float cap_exact(const CapArgs& r, float s) {
  float q;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + ex2_mufu(s * r.k2)));
  return fmaf(-2.f * r.unit, q, r.unit);
}
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
// A pair within the cap, over s; then the pair itself, and with something added.
__device__ __forceinline__ float2 cap_part(const CapArgs& r, float2 s) {
  const float2 u = fmul2(s, s);
  float2 p = ffma2(u, r.a[5], r.a[4]);
  p = ffma2(u, p, r.a[3]);
  p = ffma2(u, p, r.a[2]);
  p = ffma2(u, p, r.a[1]);
  return ffma2(u, p, r.a[0]);
}
// Up to half of the cap.
__device__ __forceinline__ float2 cap_half_part(const CapArgs& r, float2 s) {
  const float2 u = fmul2(s, s);
  float2 p = ffma2(u, r.b[3], r.b[2]);
  p = ffma2(u, p, r.b[1]);
  return ffma2(u, p, r.b[0]);
}
__device__ __forceinline__ float2 cap_half(const CapArgs& r, float2 s, float2 plus) { return ffma2(s, cap_half_part(r, s), plus); }
__device__ __forceinline__ float2 cap_pair(const CapArgs& r, float2 s) { return fmul2(s, cap_part(r, s)); }
__device__ __forceinline__ float2 cap_pair(const CapArgs& r, float2 s, float2 plus) { return ffma2(s, cap_part(r, s), plus); }
// The same of numbers that are parts of the cap already, tanh(x).
__device__ __forceinline__ float2 tanh_pair(float2 x) {
  const float2 u = fmul2(x, x);
  constexpr float C0 = CAP_C[0], C1 = CAP_C[1], C2 = CAP_C[2], C3 = CAP_C[3], C4 = CAP_C[4], C5 = CAP_C[5];
  float2 p = ffma2(u, splat(C5), splat(C4));
  p = ffma2(u, p, splat(C3));
  p = ffma2(u, p, splat(C2));
  p = ffma2(u, p, splat(C1));
  return fmul2(x, ffma2(u, p, splat(C0)));
}
__device__ __forceinline__ float tanh_exact(float x) {
  float q;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + ex2_mufu(x * 2.8853900817779268f)));
  return fmaf(-2.f, q, 1.f);
}
// tanh in 16 bits from which both t and 1 - t^2 come with 11 bits. A t near to 1 has lost its distance to 1 when it is rounded (5 % of the derivative at x = 3, all of it from 4.5 on). So
// up to t = tanh(1) the code is t, and beyond it K / sqrt(1 - |t|), which goes on from there: t is off by 2^-11 of itself below and by 2^-10 (1 - |t|) above, the derivative
// by 2^-11 2 t^2 / (1 - t^2) <= 2^-9.5 below and 2^-10 above, relative, up to |x| = 12.4, whose derivative of 6.4e-11 is all beyond it have.
constexpr float CAP_BEND = 0.76159416f, CAP_BEND_K = 0.37186221f, CAP_CODE_MOST = 65504.f;
__device__ __forceinline__ float tanh_coded(float x, float& code) {
  const float a = fabsf(x);
  float q, k;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + ex2_mufu(a * 2.8853900817779268f)));
  const float far = 2.f * q, t = copysignf(1.f - far, x);   // far: 1 - |t|
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(k) : "f"(far));
  code = a <= 1.f ? t : copysignf(fminf(CAP_BEND_K * k, CAP_CODE_MOST), x);
  return t;
}
__device__ __forceinline__ float tanh_decoded(float code, float& slope) {
  const float a = fabsf(code);
  float q;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(a));
  q *= CAP_BEND_K;
  const float far = q * q;
  const bool below = a <= CAP_BEND;
  slope = below ? fmaf(-code, code, 1.f) : far * (2.f - far);
  return below ? code : copysignf(1.f - far, code);
}
// A warp's numbers in tensor memory, n x 16 columns of its lanes, capped in place by the exact form. A loop of its own, so that the polynomial's code is all that
// tiles within the cap fetch.
__device__ __forceinline__ void cap_in_place(const CapArgs& r, uint32_t taddr, int n) {
#pragma unroll 1
  for (int c = 0; c < n; ++c) {
    uint32_t v[16];
    tmem_ld_32x16(taddr + c * 16, v);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(cap_exact(r, __uint_as_float(v[i])));
    tmem_st_32x16(taddr + c * 16, v);
  }
  tmem_st_wait();
}

}  // namespace mtb
