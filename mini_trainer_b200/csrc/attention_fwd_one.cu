// Varlen causal GQA attention forward, one query tile per CTA: the kernel is in attention_fwd_one.cuh.
#include "attention_fwd_one.cuh"

// plan: query-block work table [n_items, 3] = (seq_start, seq_len, q0), blocks of 128 rows, most work first.
extern "C" int mtb200_attn_fwd_one(const void* qkv, long long ld, void* out, long long ldo, float* lse, const int* plan, int n_items,
                                   int T, int Hq, int Hkv, int D, float scale, int* status, cudaStream_t st) {
  using namespace mtb;
  using namespace mtb::att_one;
  if (n_items <= 0 || T <= 0) return 0;
  const Params<NoRule> p{reinterpret_cast<__nv_bfloat16*>(out), ldo, lse, plan, T, Hq, Hkv, scale, status, {}};
  return fwd_one<NoRule>(qkv, ld, ldo, T, n_items, D, p, st);
}
