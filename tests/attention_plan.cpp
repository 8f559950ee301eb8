// The attention's split of its work, for a test without a GPU.
#include "../metallix_amd/csrc/mxs_attention_plan.h"

extern "C" void plan(const uint32_t* in, uint32_t* out) {
  const mxs::AttPlan p = mxs::attention_plan(in[0], in[1], in[2], in[3], in[4], in[5], in[6], in[7]);
  const uint32_t v[10] = {p.dp, p.rb, p.wq, p.small, p.sp, p.ss, p.slots, p.ng, p.wb, p.nt};
  for (int i = 0; i < 10; ++i) out[i] = v[i];
}
extern "C" uint64_t bytes(uint64_t queries, uint32_t slots, uint32_t dp) { return mxs::att_bytes(queries, slots, dp); }
