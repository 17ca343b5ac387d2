// The argument checks of the paged decode ops and the layout of a value's codes
// (csrc/decode_checks.hpp, paged_layout.hpp) behind C functions, for the CPU
// tests: pointers are numbers here and are never followed.
#include "../../atlas_amd/csrc/decode_checks.hpp"

namespace {
template <typename T>
T* at(uint64_t address) {
    return reinterpret_cast<T*>(address);
}
}  // namespace

#define CACHE_PARAMS                                                                                                    \
    int format, uint64_t pages, uint64_t table, uint32_t page_count, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, \
        uint32_t sequences, uint32_t table_width
#define CACHE {at<uint8_t>(pages), at<uint32_t>(table), page_count, page_size, kv_heads, head_dim, sequences, table_width, format}

extern "C" {

uint64_t paged_bytes(CACHE_PARAMS) { return atlas::paged_pool_bytes(CACHE); }
uint32_t value_place(uint32_t head_dim, uint32_t dim) { return atlas::paged_value_place(head_dim, dim); }

const char* check_append(CACHE_PARAMS, uint64_t key, uint64_t value, uint64_t query, uint64_t query_out, uint64_t cosine,
                         uint64_t sine, uint64_t ids, uint64_t positions, uint32_t rope_rows, uint32_t rope_stride,
                         uint32_t tokens, uint32_t q_heads) {
    return atlas::paged_append_error({CACHE, at<float>(key), at<float>(value), at<float>(query), at<float>(query_out),
                                      at<float>(cosine), at<float>(sine), at<uint32_t>(ids), at<uint32_t>(positions), rope_rows,
                                      rope_stride, tokens, q_heads});
}

const char* check_read(CACHE_PARAMS, uint64_t ids, uint64_t positions, uint64_t key, uint64_t value, uint32_t rows) {
    return atlas::paged_read_error({CACHE, at<uint32_t>(ids), at<uint32_t>(positions), at<float>(key), at<float>(value), rows});
}

const char* check_attention(CACHE_PARAMS, uint64_t q, uint64_t lengths, uint64_t output, uint32_t q_heads, uint32_t window,
                            float scale, uint64_t workspace) {
    return atlas::paged_attention_error(
        {CACHE, at<float>(q), at<uint32_t>(lengths), at<float>(output), q_heads, window, scale, at<void>(workspace)});
}

const char* check_logprobs(uint64_t logits, uint64_t row_stride, uint64_t tokens, uint64_t logprobs, uint64_t entropy,
                           uint64_t top_ids, uint64_t top_logprobs, uint32_t rows, uint32_t vocab, uint32_t given, uint32_t top,
                           double inv_temperature, uint64_t workspace) {
    return atlas::token_logprobs_error({at<float>(logits), row_stride, at<uint32_t>(tokens), at<float>(logprobs),
                                        at<float>(entropy), at<uint32_t>(top_ids), at<float>(top_logprobs), rows, vocab, given,
                                        top, inv_temperature, at<void>(workspace)});
}
}
