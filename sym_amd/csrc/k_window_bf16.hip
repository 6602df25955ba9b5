// k_window_bf16.hip - attention over packed sequences in bf16.
#include "k_window.h"

namespace relx {

hipError_t window_launch_bf16(const WindowArgs &a, bool back, hipStream_t s) { return window_by_width<kBF16>(a, back, s); }

} // namespace relx
