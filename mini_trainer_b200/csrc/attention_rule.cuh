// What the attention kernels do to a score between Q K^T and the softmax when they run under a rule (ops/attention_rule.py):
//   s   = scale q.k
//   s  -> cap tanh(s / cap)                        (CAP)
//   s  -> s - slope[head] |i - j|                  (BIAS; i, j: positions of query and key in their sample)
//   query i sees key j  iff  (j <= i and i - j < window) or j < prefix         (the diagonal is always seen: no row is empty)
// The kernels are instances of the same templates as the plain causal ones; NoRule compiles to what those were. Masks need no parameter of the
// template: which tiles exist, and which of them are crossed by an edge of the mask, is found per tile.
//
// tanh. For |s| <= cap (raw scores that big are rare: then the whole warp's tile takes the exact form) an odd polynomial of degree nine, fitted to the least
// relative error on [-1, 1] (6.1e-6: a twentieth of what the exponentials' cubic is off), its coefficients times powers of scale / cap, so that a pair of scores costs six
// packed instructions from the raw product to the exponential's argument where it cost one. tanh as 1 - 2 / (1 + e^2x) takes two more operations on
// the special-function unit, which bounds the softmax as it is: three times the work there.
#pragma once
#include <stdint.h>

#include "ptx.cuh"

namespace mtb {

struct AttRuleArgs {
  int window;            // keys a query sees, itself among them; 1 << 30 for all
  const float* slopes;   // [Hq]
  // scores in units of log2 e: cap2 tanh(s k), k = scale / cap
  float2 a[5];           // twice each, for packed arithmetic: polynomial in the raw product: s (a0 + a1 s^2 + ...)
  float most;            // |raw product| up to which it holds
  float cap2, k2;        // cap log2 e; 2 k log2 e
  float inv2;            // -1 / cap2^2
};

template <bool CAP_, bool BIAS_>
struct Rule { static constexpr bool ON = true, CAP = CAP_, BIAS = BIAS_; static constexpr int ROW = 4; using Args = AttRuleArgs; };   // ROW: ints of a row of the work table
struct NoRule { static constexpr bool ON = false, CAP = false, BIAS = false; static constexpr int ROW = 3; struct Args {}; };

inline AttRuleArgs att_rule_args(float scale, float cap, int window, const float* slopes) {
  AttRuleArgs r{};
  r.window = window > 0 && window < (1 << 30) ? window : 1 << 30;
  r.slopes = slopes;
  if (cap > 0.f) {
    constexpr double C[5] = {0.99999394, -0.33300744, 0.13050084, -0.0450287, 0.00914157};
    const double k = static_cast<double>(scale) / cap, c2 = static_cast<double>(cap) * 1.4426950408889634;
    double p = k;
    for (int i = 0; i < 5; ++i, p *= k * k) r.a[i].x = r.a[i].y = static_cast<float>(c2 * C[i] * p);
    r.most = static_cast<float>(1.0 / k);
    r.cap2 = static_cast<float>(c2);
    r.k2 = static_cast<float>(2.0 * k * 1.4426950408889634);
    r.inv2 = static_cast<float>(-1.0 / (c2 * c2));
  }
  return r;
}
// Range of scale / cap for which the coefficients, and the polynomial's terms wherever it is taken, are normal numbers.
inline bool att_cap_ok(float scale, float cap) { return cap == 0.f || (scale > 0.f && cap > 0.f && scale >= cap * 0x1p-13f && scale <= cap * 0x1p10f); }

// Capped score in units of log2 e, any argument: infinities saturate.
__device__ __forceinline__ float cap_exact(const AttRuleArgs& r, float s) {
  float q;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.f + ex2_mufu(s * r.k2)));
  return fmaf(-2.f * r.cap2, q, r.cap2);
}
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
// a0 + a1 s^2 + ... of a pair: times s the capped score.
__device__ __forceinline__ float2 cap_poly(const AttRuleArgs& r, float2 s) {
  const float2 u = fmul2(s, s);
  float2 p = ffma2(u, r.a[4], r.a[3]);
  p = ffma2(u, p, r.a[2]);
  p = ffma2(u, p, r.a[1]);
  return ffma2(u, p, r.a[0]);
}

// A warp's scores in tensor memory, n x 16 columns of its lanes, capped in place by the exact form. Where scores beyond the cap are, which is rare, this
// is a loop of its own, so that the polynomial's code is all that the others fetch.
__device__ __forceinline__ void cap_in_place(const AttRuleArgs& r, uint32_t taddr, int n) {
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

// Bits 0 .. n - 1.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Key tiles of 128 that a tile of query rows [q0, q0 + 128) looks at: the prefix's, then those from `skip` on behind them.
struct AttTiles {
  int prefix_tiles, skip;
  __device__ __forceinline__ int operator()(int j) const { return j >= prefix_tiles ? j + skip : j; }
};
// Whether every row of [q0, q0 + 128) sees every key of [k0, k0 + 128).
__device__ __forceinline__ bool att_all_seen(const AttRuleArgs& r, int q0, int k0, int prefix) {
  return k0 + 128 <= prefix || (k0 + 127 <= q0 && q0 + 127 - k0 < r.window);
}
// Of 32 keys from k on, the ones that query i sees.
__device__ __forceinline__ uint32_t att_keys_seen(const AttRuleArgs& r, int i, int k, int prefix) {
  return low_bits(prefix - k) | (low_bits(i + 1 - k) & ~low_bits(i + 1 - r.window - k));
}
// Of 32 queries from i on, the ones that see key j.
__device__ __forceinline__ uint32_t att_queries_seen(const AttRuleArgs& r, int j, int i, int prefix) {
  return j < prefix ? 0xffffffffu : low_bits(j + r.window - i) & ~low_bits(j - i);
}

}  // namespace mtb
