// paged_attention_f16.hip -- the paged attention of f16 pages.
#include "paged_attention.hpp"

namespace atlas {

hipError_t launch_paged_attention_f16(hipStream_t stream, const PagedAttnParams& a) { return launch_paged_format<kKvF16>(stream, a); }

}  // namespace atlas
