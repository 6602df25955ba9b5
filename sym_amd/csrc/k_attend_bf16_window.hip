// k_attend_bf16_window.hip - tree attention with bf16 queries over a cache of bf16, with a window.
#include "k_attend.h"

namespace relx {

hipError_t attend_launch_bf16_window(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  return attend_width<kWindow, kBF16, false>(a, p, s);
}

} // namespace relx
