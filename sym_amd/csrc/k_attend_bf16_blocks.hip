// k_attend_bf16_blocks.hip - tree attention with bf16 queries over a cache of int8 with a scale a block.
#include "k_attend.h"

namespace relx {

hipError_t attend_launch_bf16_blocks(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  return attend_width<kBlocks, kBF16, true>(a, p, s);
}

} // namespace relx
