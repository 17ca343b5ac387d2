// decode_checks.hpp -- the argument checks of the shared-prompt and the paged
// decode ops, on the host and without a device: each gives what is wrong, or null.
#pragma once

#include "launch.hpp"
#include "paged_plan.hpp"

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

// The kernels take a scale with log2(e) in it, which has to be a number of f32 still.
inline const char* attention_scale_error(float scale) {
    return std::isfinite(scale * 1.44269504f) ? nullptr : "attention scale must be finite, and at most 2.3e38";
}

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
    if (const char* error = attention_scale_error(a.scale)) return error;
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

// Spans of any lengths that share bytes; a null span has none.
inline bool spans_overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + b_bytes && y < x + a_bytes;
}

inline const char* paged_cache_sizes_error(const PagedCache& c) {
    if (c.format != kKvF32 && c.format != kKvF16 && c.format != kKvQ8_0 && c.format != kKvQ4_0) return "unknown cache format";
    if (c.page_size < 16 || c.page_size > 4096 || (c.page_size & (c.page_size - 1)) != 0)
        return "a page has a power of two of rows, 16 to 4096";
    if (c.head_dim == 0 || c.head_dim > 256 || c.head_dim % (c.format == kKvF32 ? 4 : c.format == kKvF16 ? 8 : 32) != 0)
        return "paged head_dim must be at most 256 and a multiple of 4 (f32), 8 (f16) or 32 (quantised)";
    if (c.kv_heads == 0 || static_cast<uint64_t>(c.kv_heads) * c.head_dim > 32768)
        return "paged caches have 1 to 32768 values a position";
    if (c.page_count == 0 || c.page_count == 0xffffffffu) return "a paged cache has 1 to 2^32 - 2 pages";
    if (c.sequences == 0 || c.sequences > kMostSequences || c.table_width == 0 ||
        static_cast<uint64_t>(c.table_width) * c.page_size > kMostPositions)
        return "paged tables have 1 to 2^20 sequences of at most 2^29 positions";
    return nullptr;
}

inline const char* paged_cache_error(const PagedCache& c) {
    if (const char* error = paged_cache_sizes_error(c)) return error;
    if (!c.pages || !c.table) return "paged cache pages or table are null";
    if (misaligned(c.pages, 16) || misaligned(c.table, 4)) return "pages must be 16-byte aligned, their table 4-byte";
    return nullptr;
}

inline uint64_t paged_pool_bytes(const PagedCache& c) { return c.page_count * paged_page_bytes(c); }

// Rows of heads that a launch holds: at most 64 lanes each.
constexpr uint64_t kMostPagedRows = 4ull * kMostGroups;

inline const char* paged_append_error(const PagedAppendArgs& a) {
    if (const char* error = paged_cache_error(a.cache)) return error;
    const PagedCache& c = a.cache;
    if (!a.key || !a.value || !a.positions) return "paged append buffer is null";
    if (a.tokens == 0) return "paged append needs tokens";
    if (!a.sequences && a.tokens > c.sequences) return "more tokens than sequences without sequence numbers";
    if (!a.cosine != !a.sine) return "rotation needs cosines and sines";
    if (a.query && (!a.cosine || !a.query_out || a.q_heads == 0)) return "a query is rotated: it needs heads, tables and an output";
    if (!a.query && a.query_out) return "query_out without a query";
    if (a.cosine && (a.rope_stride < c.head_dim / 2 || a.rope_rows < c.table_width * c.page_size))
        return "rotation tables need head_dim / 2 values for every position of the table";
    const uint64_t heads = a.query ? a.q_heads : 0;
    if (a.tokens * (heads + 2ull * c.kv_heads) > kMostPagedRows) return "paged append has more than 2^25 rows of heads";
    if (misaligned(a.key, 16) || misaligned(a.value, 16) || misaligned(a.query, 16) || misaligned(a.query_out, 16))
        return "paged append keys, values and queries must be 16-byte aligned";
    if (misaligned(a.cosine, 4) || misaligned(a.sine, 4) || misaligned(a.sequences, 4) || misaligned(a.positions, 4))
        return "paged append tables, sequences and positions must be 4-byte aligned";
    const uint64_t pool = paged_pool_bytes(c), row = 4ull * a.tokens * c.head_dim, kv = row * c.kv_heads, q = row * heads;
    if (a.query && a.query != a.query_out && spans_overlap(a.query, q, a.query_out, q)) return "query_out must be query or not overlap it";
    if (spans_overlap(c.pages, pool, a.key, kv) || spans_overlap(c.pages, pool, a.value, kv) ||
        spans_overlap(c.pages, pool, a.query, q) || spans_overlap(c.pages, pool, a.query_out, q) ||
        spans_overlap(a.query_out, q, a.key, kv) || spans_overlap(a.query_out, q, a.value, kv))
        return "paged append outputs overlap its inputs";
    return nullptr;
}

inline const char* paged_read_error(const PagedReadArgs& a) {
    if (const char* error = paged_cache_error(a.cache)) return error;
    const PagedCache& c = a.cache;
    if ((!a.key && !a.value) || !a.positions) return "paged read buffer is null";
    if (a.rows == 0) return "paged read needs rows";
    if (!a.sequences && a.rows > c.sequences) return "more rows than sequences without sequence numbers";
    if (a.rows * (2ull * c.kv_heads) > kMostPagedRows) return "paged read has more than 2^25 rows of heads";
    if (misaligned(a.key, 16) || misaligned(a.value, 16)) return "paged read outputs must be 16-byte aligned";
    if (misaligned(a.sequences, 4) || misaligned(a.positions, 4)) return "paged read sequences and positions must be 4-byte aligned";
    const uint64_t pool = paged_pool_bytes(c), out = 4ull * a.rows * c.kv_heads * c.head_dim;
    if (spans_overlap(c.pages, pool, a.key, out) || spans_overlap(c.pages, pool, a.value, out) ||
        spans_overlap(a.key, out, a.value, out))
        return "paged read outputs overlap";
    return nullptr;
}

// Of all rows of up to 16 query heads: a part has 1024 units of 16 positions, and there are 2^20 parts.
constexpr uint64_t kMostPagedPositions = 1ull << 34;

inline const char* paged_attention_sizes_error(const PagedCache& c, uint32_t q_heads) {
    if (const char* error = paged_cache_sizes_error(c)) return error;
    if (q_heads == 0 || q_heads % c.kv_heads != 0) return "paged attention needs q_heads a multiple of kv_heads";
    if (static_cast<uint64_t>(c.sequences) * q_heads > kMostGroups) return "paged attention has more than 2^23 query rows";
    const uint64_t rows = static_cast<uint64_t>(c.sequences) * c.kv_heads * ((q_heads / c.kv_heads + 15) / 16);
    if (static_cast<uint64_t>(c.table_width) * c.page_size * rows > kMostPagedPositions)
        return "paged attention is limited to 2^34 positions of all sequences and KV heads together";
    return nullptr;
}

inline const char* paged_attention_error(const PagedAttentionArgs& a) {
    if (const char* error = paged_cache_error(a.cache)) return error;
    if (const char* error = paged_attention_sizes_error(a.cache, a.q_heads)) return error;
    if (!a.q || !a.lengths || !a.output || !a.workspace) return "paged attention buffer is null";
    if (const char* error = attention_scale_error(a.scale)) return error;
    if (misaligned(a.q, 16) || misaligned(a.output, 16) || misaligned(a.workspace, 16) || misaligned(a.lengths, 4))
        return "paged attention q, output and workspace must be 16-byte aligned, lengths 4-byte";
    const uint64_t bytes = 4ull * a.cache.sequences * a.q_heads * a.cache.head_dim;
    if (spans_overlap(a.q, bytes, a.output, bytes) || spans_overlap(a.cache.pages, paged_pool_bytes(a.cache), a.output, bytes))
        return "paged attention output overlaps q or the pages";
    // the second launch goes by what the first left in the workspace, and by the lengths that it went by
    const struct {
        const void* at;
        uint64_t bytes;
    } inputs[] = {{a.q, bytes},
                  {a.cache.pages, paged_pool_bytes(a.cache)},
                  {a.lengths, 4ull * a.cache.sequences},
                  {a.cache.table, 4ull * a.cache.sequences * a.cache.table_width}};
    const uint64_t room = paged_attention_workspace(a.cache, a.q_heads);
    if (spans_overlap(a.output, bytes, a.workspace, room)) return "paged attention output overlaps the workspace";
    for (const auto& x : inputs)
        if (spans_overlap(x.at, x.bytes, a.workspace, room) || spans_overlap(x.at, x.bytes, a.output, bytes))
            return "paged attention output or workspace overlaps its inputs";
    return nullptr;
}

inline const char* token_logprobs_sizes_error(uint32_t rows, uint32_t vocab, uint32_t top) {
    if (rows == 0 || vocab == 0) return "log probabilities need rows and a vocabulary";
    if (vocab > kMostPositions || top > kMostTop) return "log probabilities are limited to 2^29 logits a row and 64 likeliest tokens";
    if ((static_cast<uint64_t>(vocab) + 4095) / 4096 * rows > kMostGroups) return "log probabilities of too many logits";
    return nullptr;
}

inline const char* token_logprobs_error(const TokenLogprobsArgs& a) {
    if (const char* error = token_logprobs_sizes_error(a.rows, a.vocab, a.top)) return error;
    if (!a.logits || !a.workspace || (a.given && (!a.tokens || !a.logprobs)) || (a.top && (!a.top_ids || !a.top_logprobs)))
        return "log probability buffer is null";
    if (a.given == 0 && a.top == 0 && !a.entropy) return "no log probabilities asked for";
    // a thread counts to `given` and a workgroup further, in 32 bits
    if (a.given > kMostPositions) return "log probabilities are limited to 2^29 given tokens a row";
    if (a.row_stride < a.vocab) return "rows of logits overlap";
    if (!std::isfinite(a.inv_temperature) || !(a.inv_temperature > 0.0)) return "inv_temperature must be finite and positive";
    if (misaligned(a.logits, 4) || misaligned(a.tokens, 4) || misaligned(a.logprobs, 4) || misaligned(a.entropy, 4) ||
        misaligned(a.top_ids, 4) || misaligned(a.top_logprobs, 4))
        return "log probability buffers must be 4-byte aligned";
    if (misaligned(a.workspace, 16)) return "log probability workspace must be 16-byte aligned";
    return nullptr;
}

}  // namespace atlas
