// paged_attention_q4_0.hip -- the paged attention of q4_0 pages.
#include "paged_attention.hpp"

namespace atlas {

hipError_t launch_paged_attention_q4_0(hipStream_t stream, const PagedAttnParams& a) { return launch_paged_format<kKvQ4_0>(stream, a); }

}  // namespace atlas
