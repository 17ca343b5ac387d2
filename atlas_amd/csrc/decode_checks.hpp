// decode_checks.hpp -- the argument checks of the shared-prompt decode ops, on
// the host and without a device: each gives what is wrong, or null.
#pragma once

#include "launch.hpp"

#include <cmath>
#include <limits>

namespace atlas {

inline uint64_t kv_row_bytes(int format, uint32_t width) {
    if (format == kKvF32) return static_cast<uint64_t>(width) * 4;
    return static_cast<uint64_t>(width / 32) * (format == kKvQ8_0 ? 34 : 18);
}

// Spans that share bytes.
inline bool overlaps(const void* a, const void* b, uint64_t bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + bytes && y < x + bytes;
}

inline bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

constexpr uint32_t kMostPositions = 1u << 29;  // of one cache, or logits of a row
constexpr uint32_t kMostSequences = 1u << 20;
// A launch has less than 2^32 threads: 256 of them to each of these.
constexpr uint32_t kMostGroups = 1u << 23;

inline const char* prefix_attention_sizes_error(const PrefixAttentionArgs& a) {
    if (a.format != kKvF32 && a.format != kKvQ8_0 && a.format != kKvQ4_0) return "unknown cache format";
    if (a.sequences == 0 || a.tokens == 0 || a.q_heads == 0 || a.kv_heads == 0 || a.q_heads % a.kv_heads != 0)
        return "prefix attention needs sequences, tokens and q_heads a multiple of kv_heads";
    if (a.head_dim == 0 || a.head_dim > 256 || a.head_dim % (a.format == kKvF32 ? 4 : 32) != 0)
        return "prefix attention head_dim must be at most 256 and a multiple of 4 (f32) or 32 (quantised)";
    if (a.prefix_length == 0 && a.capacity == 0) return "prefix attention has neither prompt nor own rows";
    if (a.prefix_length > kMostPositions || a.capacity > kMostPositions ||
        static_cast<uint64_t>(a.sequences) * a.capacity > std::numeric_limits<uint32_t>::max())
        return "prefix attention cache positions overflow";
    const uint64_t rows = static_cast<uint64_t>(a.sequences) * a.tokens;
    if (rows > kMostGroups || rows * a.q_heads > kMostGroups) return "prefix attention has more than 2^23 query rows";
    if (static_cast<uint64_t>(a.kv_heads) * a.head_dim > 32768) return "prefix attention cache rows are limited to 32768 values";
    return nullptr;
}

inline const char* prefix_attention_error(const PrefixAttentionArgs& a) {
    if (const char* error = prefix_attention_sizes_error(a)) return error;
    if (!a.q || !a.output || !a.workspace) return "prefix attention buffer is null";
    if (a.prefix_length && !a.prefix) return "prefix attention prompt cache is null";
    if (a.prefix_length > a.prefix_capacity) return "prefix_length exceeds prefix_capacity";
    if (a.capacity && (!a.cache || !a.lengths)) return "prefix attention own cache or lengths are null";
    if (a.weights_out && !a.capacity) return "attention weights need own rows";
    if (a.weights_in && !a.weights_out) return "weights_in without weights_out";
    if (!std::isfinite(a.scale)) return "attention scale must be finite";
    if (misaligned(a.q, 16) || misaligned(a.output, 16) || misaligned(a.workspace, 16))
        return "prefix attention q, output and workspace must be 16-byte aligned";
    const uintptr_t to = a.format == kKvF32 ? 16 : 2;
    if ((a.prefix_length && misaligned(a.prefix, to)) || (a.capacity && misaligned(a.cache, to)))
        return "prefix attention caches must be 16-byte (f32) or 2-byte (quantised) aligned";
    if (misaligned(a.weights_in, 4) || misaligned(a.weights_out, 4) || misaligned(a.lengths, 4))
        return "attention weights and lengths must be 4-byte aligned";
    if (overlaps(a.q, a.output, 4ull * a.sequences * a.tokens * a.q_heads * a.head_dim))
        return "prefix attention output overlaps q";
    if (a.weights_in && a.weights_in != a.weights_out && overlaps(a.weights_in, a.weights_out, 4ull * a.sequences * a.capacity))
        return "weights_in and weights_out overlap";
    return nullptr;
}

inline const char* kv_evict_error(const KvEvictArgs& a, int format, uint32_t kv_width) {
    if (!a.cache || !a.cache_out || !a.weights || !a.weights_out || !a.lengths || !a.lengths_out || !a.kept)
        return "KV evict buffer is null";
    if (a.sequences == 0 || a.capacity == 0 || kv_width == 0 || kv_width > 32768 || a.sequences > kMostSequences ||
        a.capacity > kMostPositions ||
        static_cast<uint64_t>(a.sequences) * a.capacity > std::numeric_limits<uint32_t>::max())
        return "KV evict dimensions are invalid (sequences * capacity below 2^32, at most 2^20 sequences, kv_width 1..32768)";
    if (a.budget == 0 || a.budget > a.capacity || a.recent > a.budget)
        return "KV evict needs recent <= budget and 1 <= budget <= capacity";
    if (format != kKvF32 && kv_width % 32 != 0) return "quantized KV rows need kv_width % 32 == 0";
    const uintptr_t to = format == kKvF32 ? 4 : 2;
    if (misaligned(a.cache, to) || misaligned(a.cache_out, to) || misaligned(a.weights, 4) || misaligned(a.weights_out, 4) ||
        misaligned(a.lengths, 4) || misaligned(a.lengths_out, 4) || misaligned(a.kept, 4))
        return "KV evict buffers must be 4-byte aligned (quantised caches 2-byte)";
    const uint64_t positions = static_cast<uint64_t>(a.sequences) * a.capacity;
    if ((a.cache != a.cache_out && overlaps(a.cache, a.cache_out, 2 * positions * kv_row_bytes(format, kv_width))) ||
        (a.weights != a.weights_out && overlaps(a.weights, a.weights_out, 4 * positions)) ||
        (a.lengths != a.lengths_out && overlaps(a.lengths, a.lengths_out, 4ull * a.sequences)))
        return "KV evict outputs must be their inputs or not overlap them";
    return nullptr;
}

inline const char* verify_draft_sizes_error(uint32_t sequences, uint32_t drafts, uint32_t vocab) {
    if (sequences == 0 || vocab == 0) return "draft verification needs sequences and a vocabulary";
    if (drafts > 1024 || vocab > kMostPositions || sequences > kMostSequences)
        return "draft verification is limited to 1024 drafts, 2^29 logits a row and 2^20 sequences";
    const uint64_t groups = (static_cast<uint64_t>(vocab) + 4095) / 4096;  // a wavefront 1024 logits
    if (groups * (2ull * drafts + 1) * sequences > kMostGroups) return "draft verification has too many logits";
    return nullptr;
}

inline const char* verify_draft_error(const VerifyDraftArgs& a) {
    if (const char* error = verify_draft_sizes_error(a.sequences, a.drafts, a.vocab)) return error;
    if (!a.target || !a.sample_uniform || !a.accepted || !a.tokens || !a.workspace ||
        (a.drafts && (!a.draft_tokens || !a.accept_uniform)))
        return "draft verification buffer is null";
    if (!std::isfinite(a.inv_temperature) || !(a.inv_temperature > 0.0)) return "inv_temperature must be finite and positive";
    if (misaligned(a.target, 4) || misaligned(a.draft, 4) || misaligned(a.draft_tokens, 4) || misaligned(a.draft_lengths, 4) ||
        misaligned(a.accept_uniform, 4) || misaligned(a.sample_uniform, 4) || misaligned(a.accepted, 4) ||
        misaligned(a.tokens, 4))
        return "draft verification buffers must be 4-byte aligned";
    if (misaligned(a.workspace, 16)) return "draft verification workspace must be 16-byte aligned";
    return nullptr;
}

}  // namespace atlas
