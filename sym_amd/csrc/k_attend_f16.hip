// k_attend_f16.hip - tree attention with f16 queries over a cache of f16.
#include "k_attend.h"

namespace relx {

hipError_t attend_launch_f16(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  return attend_width<kF16, false>(a, p, s);
}

} // namespace relx
