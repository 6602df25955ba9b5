// k_attend_f16_window.hip - tree attention with f16 queries over a cache of f16, with a window.
#include "k_attend.h"

namespace relx {

hipError_t attend_launch_f16_window(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  return attend_width<kWindow, kF16, false>(a, p, s);
}

} // namespace relx
