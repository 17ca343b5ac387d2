// paged_layout.hpp -- the layout of a cache in pages.
//
// A pool is [page][K | V][KV head][part]: a head's rows of a page lie together,
// so that whoever attends with one head reads whole lines.  A part has
// page_size (a power of two, 16 at least) rows of head_dim values:
//   f32, f16   [row][head_dim]
//   Q8_0, Q4_0 the codes, [row][head_dim or head_dim / 2 bytes], then the
//              scales, f16 [row / 4][block][row % 4], a block being 32 values.
// Codes and scales apart, everything lies on its own alignment (blocks of 34 and
// 18 bytes do not), and the scales of a lane's four keys of an MFMA result are
// one load.  Q4_0 codes are two to a byte, the first one low; a value is
// (code - 8) * scale.  A key's codes are in the order of its dims.  A value's are
// in the order in which the product over keys wants them: lane i of sixteen has
// dims 32 b + 2 i and 32 b + 2 i + 1 of every block b, and loads them at once.
// Its blocks are taken in runs of 8, 4, 2 and 1 (the binary digits of head_dim / 32,
// the largest first), a run being [16][block][2] codes: any number of blocks,
// every load aligned.
#pragma once

#include "launch.hpp"

namespace atlas {

__host__ __device__ inline uint32_t paged_row_code_bytes(int format, uint32_t head_dim) {
    switch (format) {
        case kKvF32: return head_dim * 4;
        case kKvF16: return head_dim * 2;
        case kKvQ8_0: return head_dim;
        default: return head_dim / 2;
    }
}
__host__ __device__ constexpr bool paged_quantised(int format) { return format == kKvQ8_0 || format == kKvQ4_0; }
// A head's rows of K or V in a page.
__host__ __device__ inline uint32_t paged_part_bytes(int format, uint32_t page_size, uint32_t head_dim) {
    return page_size * (paged_row_code_bytes(format, head_dim) + (paged_quantised(format) ? head_dim / 32 * 2 : 0));
}
__host__ __device__ inline uint64_t paged_page_bytes(const PagedCache& c) {
    return 2ull * c.kv_heads * paged_part_bytes(c.format, c.page_size, c.head_dim);
}

// The first block of the run that holds block b of `blocks`, and the run's length.
__host__ __device__ inline void paged_run(uint32_t blocks, uint32_t b, uint32_t& first, uint32_t& length) {
    first = 0;
    length = 8;
    // head_dim is at most 256: 8 blocks
    while (!(blocks & length) || b >= first + length) {
        if (blocks & length) first += length;
        length /= 2;
    }
}
// Where the codes of dims d and d + 1 (d even) of a value start.
__host__ __device__ inline uint32_t paged_value_place(uint32_t head_dim, uint32_t d) {
    uint32_t first, length;
    paged_run(head_dim / 32, d / 32, first, length);
    return 32 * first + (d % 32 / 2) * 2 * length + 2 * (d / 32 - first);
}

}  // namespace atlas
