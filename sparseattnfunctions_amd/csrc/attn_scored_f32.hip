// Attention with score rules: the kernels of fp32 operands.
#include "attn_scored_pass.h"

void sa_scored::launch_pass_f32(const ScoredArgs& a, const MergeArgs& m, const PassCall& c) {
  launch_pass_of<float>(a, m, c);
}
