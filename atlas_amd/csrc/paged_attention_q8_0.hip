// paged_attention_q8_0.hip -- the paged attention of q8_0 pages.
#include "paged_attention.hpp"

namespace atlas {

hipError_t launch_paged_attention_q8_0(hipStream_t stream, const PagedAttnParams& a) { return launch_paged_format<kKvQ8_0>(stream, a); }

}  // namespace atlas
