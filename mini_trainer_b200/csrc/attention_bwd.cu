// Varlen causal GQA attention backward: the kernels are in attention_bwd.cuh.
#include "attention_bwd.cuh"

// plan: key-block work table [n_items, 3] = (seq_start, seq_len, k0), most work first.
// dq_acc: fp32 [T, Hq*D] scratch, 16-byte aligned; delta: fp32 [Hq, T] scratch.
// splits: CTAs that share the query heads of a key block; more than one needs counters, an epoch and scratch as the split-K GEMM does.
// in_order: the kernel is launched behind its predecessor's end (launch_bwd).
extern "C" int mtb200_attn_bwd(const void* qkv, long long ld, const void* out, long long ldo, const void* dout, long long lddo,
                               void* dqkv, long long ldq, const float* lse, float* delta, float* dq_acc, const int* plan,
                               int n_items, int T, int Hq, int Hkv, int D, int splits, unsigned long long* counters, unsigned long long epoch, float* part, long long part_bytes, float scale, int in_order, int* status, cudaStream_t st) {
  using namespace mtb;
  if (n_items <= 0 || T <= 0) return 0;
  if (Hkv <= 0) return -10;
  const AttBwdParams<NoRule> p{reinterpret_cast<__nv_bfloat16*>(dqkv), ldq, lse, delta, dq_acc, plan, T, Hq, Hkv, Hq / Hkv, 0xffffffffu / static_cast<unsigned>(Hkv), splits,
                       part, counters, epoch, scale, status, {}};
  return bwd<NoRule>(qkv, ld, out, ldo, dout, lddo, T, n_items, D, part_bytes, in_order != 0, delta, p, st);
}
