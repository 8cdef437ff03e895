// Prefill attention over FP8 pages.
#include "paged_prefill.h"

namespace vfkv {
hipError_t launch_paged_prefill_byte(const PagedAttnLaunch& L, hipStream_t stream) { return launch_prefill_of<kF8>(L, stream); }
}  // namespace vfkv
