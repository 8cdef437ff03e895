// Prefill attention over F32 pages.
#include "paged_prefill.h"

namespace vfkv {
hipError_t launch_paged_prefill_full(const PagedAttnLaunch& L, hipStream_t stream) { return launch_prefill_of<kF32>(L, stream); }
}  // namespace vfkv
