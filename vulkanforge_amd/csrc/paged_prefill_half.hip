// Prefill attention over F16 pages.
#include "paged_prefill.h"

namespace vfkv {
hipError_t launch_paged_prefill_half(const PagedAttnLaunch& L, hipStream_t stream) { return launch_prefill_of<kF16>(L, stream); }
}  // namespace vfkv
