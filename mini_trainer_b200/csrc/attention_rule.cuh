// What the attention kernels do to a score between Q K^T and the softmax when they run under a rule (ops/attention_rule.py):
//   s   = scale q.k
//   s  -> cap tanh(s / cap)                        (CAP)
//   s  -> s - slope[head] |i - j|                  (BIAS; i, j: positions of query and key in their sample)
//   query i sees key j  iff  (j <= i and i - j < window) or j < prefix         (the diagonal is always seen: no row is empty)
// The kernels are instances of the same templates as the plain causal ones; NoRule compiles to what those were. Masks need no parameter of the
// template: which tiles exist, and which of them are crossed by an edge of the mask, is found per tile.
// The cap is in cap.cuh.
#pragma once
#include <stdint.h>

#include "cap.cuh"
#include "ptx.cuh"

namespace mtb {

struct AttRuleArgs {
  int window;            // keys a query sees, itself among them; 1 << 30 for all
  const float* slopes;   // [Hq]
  CapArgs cap;           // of raw products
};

template <bool CAP_, bool BIAS_>
struct Rule { static constexpr bool ON = true, CAP = CAP_, BIAS = BIAS_; static constexpr int ROW = 4; using Args = AttRuleArgs; };   // ROW: ints of a row of the work table
struct NoRule { static constexpr bool ON = false, CAP = false, BIAS = false; static constexpr int ROW = 3; struct Args {}; };

inline AttRuleArgs att_rule_args(float scale, float cap, int window, const float* slopes) {
  AttRuleArgs r{};
  r.window = window > 0 && window < (1 << 30) ? window : 1 << 30;
  r.slopes = slopes;
  if (cap > 0.f) r.cap = cap_args(scale, cap, static_cast<double>(cap) * 1.4426950408889634);
  return r;
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


// Scores of one query and C x 32 keys from `key` on, formed in place, and their maximum. EDGE: an edge of the mask crosses the tile; masked scores become -inf, `seen` and `any`
// (whether one of the warp's rows sees a key of 32) are left for the exponentials. With a cap or a bias the scores and the maximum come in units of log2 e
// (FORM); without either they stay products, which the scale still has to be applied to. taddr: where the products came from in tensor memory.
template <class R, bool EDGE, int C>
__device__ __forceinline__ float att_form(const AttRuleArgs& r, uint32_t (&sv)[C][32], uint32_t (&seen)[C], bool (&any)[C], int query, int key, int prefix, bool right,
                                          float slope2, float2 sl2v, uint32_t taddr) {
  auto pair = [&](int c, int i) { return make_float2(__uint_as_float(sv[c][2 * i]), __uint_as_float(sv[c][2 * i + 1])); };
  auto put = [&](int c, int i, float2 v) { sv[c][2 * i] = __float_as_uint(v.x); sv[c][2 * i + 1] = __float_as_uint(v.y); };
#pragma unroll
  for (int c = 0; c < C; ++c) {
    seen[c] = EDGE ? att_keys_seen(r, query, key + c * 32, prefix) : 0xffffffffu;
    any[c] = !EDGE || __any_sync(0xffffffffu, seen[c] != 0u);
  }
  if constexpr (R::CAP) {
    float big = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float b = 0.f;
#pragma unroll
      for (int i = 0; i < 32; i += 2) b = fmax3(b, fabsf(__uint_as_float(sv[c][i])), fabsf(__uint_as_float(sv[c][i + 1])));
      big = fmaxf(big, b);
    }
    if (__all_sync(0xffffffffu, big <= r.cap.most)) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (EDGE && !any[c]) continue;
#pragma unroll
        for (int i = 0; i < 16; ++i) put(c, i, cap_pair(r.cap, pair(c, i)));
      }
    } else {
      cap_in_place(r.cap, taddr, 2 * C);
#pragma unroll
      for (int c = 0; c < C; ++c) tmem_ld_32x32(taddr + c * 32, sv[c]);
      tmem_ld_wait();
    }
  }
  if constexpr (R::BIAS) {
    auto add = [&](int c, int i, float2 b) { put(c, i, R::CAP ? fadd2(pair(c, i), b) : ffma2(pair(c, i), sl2v, b)); };
    const float from = static_cast<float>(key - query);
    if (right) {   // keys behind the query, which only a prefix shows it
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) add(c, i, make_float2(-slope2 * fabsf(from + (c * 32 + 2 * i)), -slope2 * fabsf(from + (c * 32 + 2 * i + 1))));
    } else {
      float2 off[4];   // within 8 keys
#pragma unroll
      for (int i = 0; i < 4; ++i) off[i] = make_float2(slope2 * (2 * i), slope2 * (2 * i + 1));
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (EDGE && !any[c]) continue;
#pragma unroll
        for (int i = 0; i < 16; ++i) add(c, i, fadd2(off[i & 3], splat(slope2 * (from + (c * 32 + (i >> 2) * 8)))));
      }
    }
  }
  float mc[C];   // independent chains
#pragma unroll
  for (int c = 0; c < C; ++c) {
    mc[c] = -INFINITY;
    if constexpr (EDGE) {
      if (!any[c]) continue;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (!(seen[c] >> i & 1u)) sv[c][i] = 0xff800000u;   // -inf
    }
    mc[c] = fmaxf(__uint_as_float(sv[c][0]), __uint_as_float(sv[c][1]));
#pragma unroll
    for (int i = 2; i < 32; i += 2) mc[c] = fmax3(mc[c], __uint_as_float(sv[c][i]), __uint_as_float(sv[c][i + 1]));
  }
  float m = fmaxf(mc[0], mc[1]);
#pragma unroll
  for (int c = 2; c < C; c += 2) m = fmax3(m, mc[c], mc[c + 1]);
  return m;
}

}  // namespace mtb
