// paged_plan.hpp -- how the attention over pages is split and launched: rules on a
// call's sizes, on the host and without a device.
#pragma once

#include "paged_layout.hpp"

namespace atlas {

inline constexpr uint32_t kPagedAttnWaves = 4;  // of a workgroup that takes a part
inline constexpr uint32_t kPagedHeads = 16;  // query heads of a row: the columns of a product

// Keys of a wavefront's step, the unit of the split: two tiles of 16 where a
// product over keys takes 32.
__host__ __device__ constexpr uint32_t paged_keys(int format) { return format == kKvF32 ? 16 : 32; }
// Workgroups to a CU.
__host__ __device__ constexpr uint32_t paged_occupancy(uint32_t head_dim) { return head_dim <= 64 ? 4 : (head_dim <= 128 ? 3 : 2); }

inline uint32_t paged_head_tiles(const PagedCache& c, uint32_t q_heads) { return (q_heads / c.kv_heads + kPagedHeads - 1) / kPagedHeads; }
inline uint64_t paged_rows(const PagedCache& c, uint32_t q_heads) {
    return static_cast<uint64_t>(c.sequences) * c.kv_heads * paged_head_tiles(c, q_heads);
}

// The first and last part of a row.
struct PagedRow {
    uint32_t first, last;
};

// Additions to a wavefront's sums in a part, a unit each: with keys alike they all round to
// one side, 2^-25 of the sum at most each.
inline constexpr uint32_t kPartUnits = 256 * kPagedAttnWaves;
inline constexpr uint32_t kMostParts = 1u << 20;

inline uint64_t round256(uint64_t v) { return (v + 255) / 256 * 256; }

struct PagedPlan {
    uint32_t few_parts, most_parts, heads;
    uint64_t out_bytes, ml_bytes, row_bytes;
};

inline PagedPlan paged_plan(const PagedCache& c, uint32_t q_heads) {
    PagedPlan p{};
    const uint32_t group = q_heads / c.kv_heads;
    p.heads = group < kPagedHeads ? group : kPagedHeads;
    const uint32_t unit = paged_keys(c.format);
    const uint64_t capacity = static_cast<uint64_t>(c.table_width) * c.page_size;
    const uint64_t rows = paged_rows(c, q_heads);
    const uint64_t units = (capacity + unit - 1) / unit * rows;
    p.few_parts = 256 * paged_occupancy(c.head_dim);
    const uint64_t long_parts = (units + kPartUnits - 1) / kPartUnits;
    uint64_t most = long_parts > p.few_parts ? long_parts : p.few_parts;
    most = most < units ? most : units;
    p.most_parts = static_cast<uint32_t>(most < kMostParts ? most : kMostParts);
    const uint64_t lines = 2ull * p.most_parts * p.heads;
    p.out_bytes = round256(lines * c.head_dim * 4);
    p.ml_bytes = round256(lines * 8);
    p.row_bytes = round256(rows * sizeof(PagedRow));
    return p;
}

inline uint64_t paged_attention_workspace(const PagedCache& c, uint32_t q_heads) {
    const PagedPlan p = paged_plan(c, q_heads);
    return p.out_bytes + p.ml_bytes + p.row_bytes;
}

inline constexpr uint32_t kFewRows = 256;  // a workgroup a CU

// The units that a row has at most, where a workgroup a row is sooner done than
// parts and their join; 0 where it is not.
//
// Of up to 256 rows by what was measured, in KB and us: a workgroup takes 48 KB/us, or
// its share of the chip's 5500; parts have the whole chip whatever the rows, but cost 4
// us more with the join, and 8 more where they are small and many.  Whole / parts, us:
// 256 windows of 512 f16 (256 dims) 30 / 52, f32 65 / 81, Q8_0 22 / 38; 64 of them f16 21
// / 30; 64 rows of up to 1024 f16 (128) 15 / 21, of 4096 49 / 31; one of 64 f32 (128) 6 /
// 10; 3 of 2048 f32 (64) 25 / 11; one of 1024 Q8_0 (256) 24 / 13.
//
// More rows are many workgroups of four wavefronts, which hide one another's beginnings
// and ends, up to 700 KB a row (400 of up to 600 f16 (256 dims) 38 / 58, 2000 of up to
// 100 Q8_0 (64) 15 / 39); the longest of longer ones ends alone (300 of up to 2000 Q8_0
// (256) 70 / 59, 512 of up to 1400 f16 110 / 108).
inline uint32_t whole_row_units(const PagedCache& c, uint32_t window, uint64_t rows) {
    const uint32_t unit = paged_keys(c.format);
    uint64_t positions = static_cast<uint64_t>(c.table_width) * c.page_size;
    if (window && window < positions) positions = window + unit;  // it may begin and end inside units
    const double row_kb = 2e-3 * positions * paged_part_bytes(c.format, c.page_size, c.head_dim) / c.page_size;
    bool whole = row_kb <= 700.0;
    if (rows <= kFewRows) {
        const double share = 5500.0 / rows;
        whole = row_kb / (share < 48.0 ? share : 48.0) < 4.0 + 8.0 * (rows < 64 ? rows / 64.0 : 1.0) + rows * row_kb / 5500.0;
        whole = whole && row_kb <= 1500.0;
    }
    whole = whole && positions <= static_cast<uint64_t>(unit) * kPartUnits;  // as many additions as in a part
    return whole ? static_cast<uint32_t>((positions + unit - 1) / unit) : 0;
}

// Wavefronts of a workgroup that takes one of few rows whole, of more than two steps for four:
// as many as the registers let stay, but six of f16 rows, whose 32 positions are twice
// the bytes (256 rows of up to 500 of 256 dims 22.6 us for 24.1 with eight, of 128 dims 11.5
// for 12.3; 100 Q8_0 rows of up to 1500 the other way, 23 for 20).
constexpr uint32_t paged_row_waves(int format, uint32_t blocks) { return blocks <= 2 ? 16 : format == kKvF16 ? 6 : 8; }
inline uint32_t paged_waves(int format, uint32_t blocks, uint32_t row_units, uint64_t rows) {
    return row_units <= 2 * kPagedAttnWaves || rows > kFewRows ? kPagedAttnWaves : paged_row_waves(format, blocks);
}

// Few rows have many parts: a workgroup for every 64 dims of one, and of 16 wavefronts; for
// every 32 where they have 128 and more (8 heads of 256 dims, 512 parts 34.1 us for 35.0; 32
// parts the other way, 13.5 for 13.9).
inline constexpr uint32_t kJoinThreads = 256, kFewThreads = 1024;
struct PagedJoin {
    uint32_t lanes, threads, groups;  // of 4 dims each; a workgroup's; workgroups of a query row
};
inline PagedJoin paged_join(const PagedCache& c, uint32_t q_heads, uint32_t most_parts) {
    const uint32_t lines = c.sequences * q_heads;
    if (lines < 64 && most_parts / paged_rows(c, q_heads) >= 128) return {8, kFewThreads, (c.head_dim + 31) / 32};
    if (lines < 512) return {16, kFewThreads, (c.head_dim + 63) / 64};
    return {c.head_dim <= 64 ? 16u : c.head_dim <= 128 ? 32u : 64u, kJoinThreads, 1};
}

}  // namespace atlas
