// Attention backward under a rule: instances of the kernel in attention_bwd.cuh (mathematics and masks: attention_rule.cuh).
#include "attention_bwd.cuh"

// Under a rule (attention_rule.cuh), as the forward was: plan [n_items, 4] = (seq_start, seq_len, k0, prefix); rows, cap, window and slopes as in mtb200_attn_rule_fwd. The first
// `whole` of the n_items Hkv key blocks have a CTA each, the others `splits`. odd: one number of device memory, zero before the first launch that is given it; number: larger than that of any
// launch before (AttRuleArgs).
extern "C" int mtb200_attn_rule_bwd(const void* qkv, long long ld, const void* out, long long ldo, const void* dout, long long lddo, void* dqkv, long long ldq,
                                    const float* lse, float* delta, float* dq_acc, const int* plan, int n_items, int T, int rows, int Hq, int Hkv, int D, int splits,
                                    unsigned long long* counters, unsigned long long epoch, float* part, long long part_bytes, float scale, float cap, int window,
                                    const float* slopes, int in_order, int whole, unsigned long long* odd, unsigned long long number, int* status, cudaStream_t st) {
  using namespace mtb;
  if (n_items <= 0 || rows <= 0) return 0;
  if (Hkv <= 0 || rows > T || !(scale > 0.f) || (cap != 0.f && !cap_ok(scale, cap)) || window < 0 || odd == nullptr || number == 0) return -10;
  AttRuleArgs args = att_rule_args(scale, cap, window, slopes);
  args.whole = whole;
  args.odd = odd;
  args.number = number;
#define BWD(C, B) bwd<Rule<C, B>>(qkv, ld, out, ldo, dout, lddo, rows, n_items, D, part_bytes, in_order != 0, delta, {reinterpret_cast<__nv_bfloat16*>(dqkv), ldq, lse, delta, dq_acc, plan, T, Hq, Hkv, Hq / Hkv, 0xffffffffu / static_cast<unsigned>(Hkv), splits, part, counters, epoch, scale, status, args}, st)
  return cap > 0.f ? (slopes ? BWD(true, true) : BWD(true, false)) : (slopes ? BWD(false, true) : BWD(false, false));
#undef BWD
}
