// k_attend_bf16.hip - tree attention with bf16 queries over a cache of bf16.
#include "k_attend.h"

namespace relx {

hipError_t attend_launch_bf16(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  return attend_width<kBF16, false>(a, p, s);
}

} // namespace relx
