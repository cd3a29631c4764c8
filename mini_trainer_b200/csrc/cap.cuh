// Numbers capped by a tanh, cap tanh(scale s / cap), in units of log2 e, as the exponentials of a softmax want them.
//
// Up to the cap (|scale s| <= cap; bigger ones are rare) an odd polynomial of degree eleven, fitted to the least relative error on [-1, 1] (5.1e-7), with the powers of
// scale / cap in its coefficients: seven packed instructions for two numbers. Beyond it tanh as 1 - 2 / (1 + e^2x), two operations on the special-function
// unit each, whose error is 2^-22 of the cap: a softmax that is bound by that unit as it is would do three times the work there.
#pragma once
#include <stdint.h>

#include "ptx.cuh"

namespace mtb {

struct CapArgs {
  float2 a[6];       // twice each, for packed arithmetic: s (a0 + a1 s^2 + ...)
  float most;        // |s| up to which that holds
  float cap2, k2;    // cap log2 e; 2 scale / cap log2 e
  float inv2;        // -1 / cap2^2: the derivative is 1 + inv2 v^2 of a capped number v
};

// Range of caps. Above it the exact form's error would pass 1e-3 of the scale's unit.
inline bool cap_ok(float scale, float cap) { return scale > 0.f && cap > 0.f && scale >= cap * 0x1p-13f && scale <= cap * 0x1p10f; }

inline CapArgs cap_args(float scale, float cap) {
  constexpr double C[6] = {0.99999949, -0.33329398, 0.13284259, -0.05168433, 0.01683263, -0.00310275};
  CapArgs r{};
  const double k = static_cast<double>(scale) / cap, c2 = static_cast<double>(cap) * 1.4426950408889634;
  double p = k;
  for (int i = 0; i < 6; ++i, p *= k * k) r.a[i].x = r.a[i].y = static_cast<float>(c2 * C[i] * p);
  r.most = k >= 0x1p-11 ? static_cast<float>(1.0 / k) : -1.f;   // below, k^11 is no normal number: the exact form throughout
  r.cap2 = static_cast<float>(c2);
  r.k2 = static_cast<float>(2.0 * k * 1.4426950408889634);
  r.inv2 = static_cast<float>(-1.0 / (c2 * c2));
  return r;
}

// Any argument: infinities saturate.
__device__ __forceinline__ float cap_exact(const CapArgs& r, float s) {
  float q;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + ex2_mufu(s * r.k2)));
  return fmaf(-2.f * r.cap2, q, r.cap2);
}
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
// A pair within the cap.
__device__ __forceinline__ float2 cap_pair(const CapArgs& r, float2 s) {
  const float2 u = fmul2(s, s);
  float2 p = ffma2(u, r.a[5], r.a[4]);
  p = ffma2(u, p, r.a[3]);
  p = ffma2(u, p, r.a[2]);
  p = ffma2(u, p, r.a[1]);
  return fmul2(s, ffma2(u, p, r.a[0]));
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
