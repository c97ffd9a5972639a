// Attention with score rules: the kernels of fp16 operands.
#include "attn_scored_pass.h"

void sa_scored::launch_pass_f16(const ScoredArgs& a, const MergeArgs& m, const PassCall& c) {
  launch_pass_of<_Float16>(a, m, c);
}
