// Attention with score rules: the kernels of bf16 operands.
#include "attn_scored_pass.h"

void sa_scored::launch_pass_bf16(const ScoredArgs& a, const MergeArgs& m, const PassCall& c) {
  launch_pass_of<__bf16>(a, m, c);
}
