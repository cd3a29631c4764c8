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
  if (cap > 0.f) r.cap = cap_args(scale, cap);
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

}  // namespace mtb
