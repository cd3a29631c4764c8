// Attention forward under a rule, one query tile per CTA: instances of the kernel in attention_fwd_one.cuh (mathematics and masks: attention_rule.cuh).
#include "attention_fwd_one.cuh"

// Arguments as of mtb200_attn_rule_fwd; plan: blocks of 128 rows.
extern "C" int mtb200_attn_rule_fwd_one(const void* qkv, long long ld, void* out, long long ldo, float* lse, const int* plan, int n_items, int T, int rows, int Hq,
                                        int Hkv, int D, float scale, float cap, int window, const float* slopes, int* status, cudaStream_t st) {
  using namespace mtb;
  using namespace mtb::att_one;
  if (n_items <= 0 || rows <= 0) return 0;
  if (rows > T || !(scale > 0.f) || (cap != 0.f && !cap_ok(scale, cap)) || window < 0) return -10;
  const AttRuleArgs args = att_rule_args(scale, cap, window, slopes);
#define FWD(C, B) fwd_one<Rule<C, B>>(qkv, ld, ldo, rows, n_items, D, {reinterpret_cast<__nv_bfloat16*>(out), ldo, lse, plan, T, Hq, Hkv, scale, status, args}, st)
  return cap > 0.f ? (slopes ? FWD(true, true) : FWD(true, false)) : (slopes ? FWD(false, true) : FWD(false, false));
#undef FWD
}
