// paged_attention_f32.hip -- the paged attention of f32 pages.
#include "paged_attention.hpp"

namespace atlas {

hipError_t launch_paged_attention_f32(hipStream_t stream, const PagedAttnParams& a) { return launch_paged_format<kKvF32>(stream, a); }

}  // namespace atlas
