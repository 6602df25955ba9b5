// k_attend_f16.hip - tree attention with f16 queries.
#include "k_attend.h"

namespace relx {

hipError_t attend_launch_f16(const AttendArgs &a, const AttendPlan &p, bool i8, hipStream_t s) {
  return i8 ? attend_width<kF16, true>(a, p, s) : attend_width<kF16, false>(a, p, s);
}

} // namespace relx
