// The argument checks of the shared-prompt decode ops (csrc/decode_checks.hpp)
// behind C functions, for the CPU tests: pointers are numbers here and are
// never followed.
#include "../../atlas_amd/csrc/decode_checks.hpp"

namespace {
template <typename T>
T* at(uint64_t address) {
    return reinterpret_cast<T*>(address);
}
}  // namespace

extern "C" {

const char* check_prefix_attention(int format, uint64_t q, uint64_t prefix, uint32_t prefix_length, uint32_t prefix_capacity,
                                   uint64_t cache, uint64_t lengths, uint32_t capacity, uint64_t output, uint64_t weights_in,
                                   uint64_t weights_out, uint32_t sequences, uint32_t tokens, uint32_t q_heads,
                                   uint32_t kv_heads, uint32_t head_dim, float scale, uint64_t workspace) {
    return atlas::prefix_attention_error({format, at<float>(q), at<uint8_t>(prefix), prefix_length, prefix_capacity,
                                          at<uint8_t>(cache), at<uint32_t>(lengths), capacity, at<float>(output),
                                          at<float>(weights_in), at<float>(weights_out), sequences, tokens, q_heads, kv_heads,
                                          head_dim, scale, at<void>(workspace)});
}

const char* check_kv_evict(int format, uint64_t cache, uint64_t cache_out, uint64_t weights, uint64_t weights_out,
                           uint64_t lengths, uint64_t lengths_out, uint64_t kept, uint32_t sequences, uint32_t capacity,
                           uint32_t kv_width, uint32_t budget, uint32_t recent) {
    return atlas::kv_evict_error({at<uint8_t>(cache), at<uint8_t>(cache_out), at<float>(weights), at<float>(weights_out),
                                  at<uint32_t>(lengths), at<uint32_t>(lengths_out), at<uint32_t>(kept), sequences, capacity, 0,
                                  budget, recent},
                                 format, kv_width);
}

const char* check_verify_draft(uint64_t target, uint64_t draft, uint64_t draft_tokens, uint64_t draft_lengths,
                               uint64_t accept, uint64_t sample, uint64_t accepted, uint64_t tokens, uint32_t sequences,
                               uint32_t drafts, uint32_t vocab, double inv_temperature, uint64_t workspace) {
    return atlas::verify_draft_error({at<float>(target), at<float>(draft), at<uint32_t>(draft_tokens),
                                      at<uint32_t>(draft_lengths), at<float>(accept), at<float>(sample), at<uint32_t>(accepted),
                                      at<uint32_t>(tokens), sequences, drafts, vocab, inv_temperature, at<void>(workspace)});
}
}
