// Attention forward under a rule, with a cap and a bias, head_dim 128: instances of attention_rule_fwd.cu.
#include "attention_fwd.cuh"

namespace mtb {
template int launch_fwd<128, Rule<true, true>>(const CUtensorMap&, const CUtensorMap&, const AttFwdParams<Rule<true, true>>&, cudaStream_t);
}  // namespace mtb
