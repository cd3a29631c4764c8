// Varlen causal GQA attention forward, pairs of query tiles: the kernel is in attention_fwd.cuh.
#include "attention_fwd.cuh"

// plan: query-block work table [n_items, 3] = (seq_start, seq_len, q0), most work first: blocks of 128 rows when Hq / Hkv is
// even, of 256 rows (row_pairs) when it is odd.
extern "C" int mtb200_attn_fwd(const void* qkv, long long ld, void* out, long long ldo, float* lse, const int* plan, int n_items,
                               int T, int Hq, int Hkv, int D, int row_pairs, float scale, int* status, cudaStream_t st) {
  using namespace mtb;
  if (n_items <= 0 || T <= 0) return 0;
  const AttFwdParams<NoRule> p{reinterpret_cast<__nv_bfloat16*>(out), ldo, lse, plan, n_items, T, Hq, Hkv, row_pairs, scale, status, {}};
  return fwd<NoRule>(qkv, ld, out, ldo, T, D, p, st);
}
