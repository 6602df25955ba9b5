// k_window_f16.hip - attention over packed sequences in f16.
#include "k_window.h"

namespace relx {

hipError_t window_launch_f16(const WindowArgs &a, bool back, hipStream_t s) { return window_by_width<kF16>(a, back, s); }

} // namespace relx
