// Attention forward under a rule, with a cap: instances of attention_rule_fwd.cu.
#include "attention_fwd.cuh"

namespace mtb {
template int launch_fwd<64, Rule<true, false>>(const CUtensorMap&, const CUtensorMap&, const AttFwdParams<Rule<true, false>>&, cudaStream_t);
template int launch_fwd<128, Rule<true, false>>(const CUtensorMap&, const CUtensorMap&, const AttFwdParams<Rule<true, false>>&, cudaStream_t);
}  // namespace mtb
