// k_attend_bf16.hip - tree attention with bf16 queries.
#include "k_attend.h"

namespace relx {

hipError_t attend_launch_bf16(const AttendArgs &a, const AttendPlan &p, bool i8, hipStream_t s) {
  return i8 ? attend_width<kBF16, true>(a, p, s) : attend_width<kBF16, false>(a, p, s);
}

} // namespace relx
