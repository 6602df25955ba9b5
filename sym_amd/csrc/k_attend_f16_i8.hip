// k_attend_f16_i8.hip - tree attention with f16 queries over a cache of int8.
#include "k_attend.h"

namespace relx {

hipError_t attend_launch_f16_i8(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  return attend_width<kWhole, kF16, true>(a, p, s);
}

} // namespace relx
