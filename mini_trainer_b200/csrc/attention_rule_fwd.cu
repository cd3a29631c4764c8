// Attention forward under a rule: instances of the kernel in attention_fwd.cuh (mathematics and masks: attention_rule.cuh).
#include "attention_fwd.cuh"

namespace mtb {
// the instances with a cap take the compiler longest: attention_rule_fwd_cap*.cu
extern template int launch_fwd<64, Rule<true, false>>(const CUtensorMap&, const CUtensorMap&, const AttFwdParams<Rule<true, false>>&, cudaStream_t);
extern template int launch_fwd<128, Rule<true, false>>(const CUtensorMap&, const CUtensorMap&, const AttFwdParams<Rule<true, false>>&, cudaStream_t);
extern template int launch_fwd<64, Rule<true, true>>(const CUtensorMap&, const CUtensorMap&, const AttFwdParams<Rule<true, true>>&, cudaStream_t);
extern template int launch_fwd<128, Rule<true, true>>(const CUtensorMap&, const CUtensorMap&, const AttFwdParams<Rule<true, true>>&, cudaStream_t);
}  // namespace mtb

// Under a rule (attention_rule.cuh). plan: [n_items, 4] = (seq_start, seq_len, q0, prefix). rows <= T: those of the samples; what lies behind them is neither
// read (the loads give zeros there) nor written. cap, window: 0 for none; slopes [Hq] fp32 or null.
extern "C" int mtb200_attn_rule_fwd(const void* qkv, long long ld, void* out, long long ldo, float* lse, const int* plan, int n_items, int T, int rows, int Hq,
                                    int Hkv, int D, int row_pairs, float scale, float cap, int window, const float* slopes, int* status, cudaStream_t st) {
  using namespace mtb;
  if (n_items <= 0 || rows <= 0) return 0;
  if (rows > T || !(scale > 0.f) || (cap != 0.f && !cap_ok(scale, cap)) || window < 0) return -10;
  const AttRuleArgs args = att_rule_args(scale, cap, window, slopes);
#define FWD(C, B) fwd<Rule<C, B>>(qkv, ld, out, ldo, rows, D, {reinterpret_cast<__nv_bfloat16*>(out), ldo, lse, plan, n_items, T, Hq, Hkv, row_pairs, scale, status, args}, st)
  return cap > 0.f ? (slopes ? FWD(true, true) : FWD(true, false)) : (slopes ? FWD(false, true) : FWD(false, false));
#undef FWD
}
