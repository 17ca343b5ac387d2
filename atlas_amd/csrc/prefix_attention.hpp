// prefix_attention.hpp -- what the kernels of the shared-prompt attention have
// in common: how lanes read the rows of a cache, and a call's parameters.
#pragma once

#include "device_common.hpp"
#include "launch.hpp"

namespace atlas {

inline constexpr int kAttnThreads = 256;
inline constexpr int kAttnWaves = kAttnThreads / kWave;
inline constexpr float kLog2e = 1.44269504088896340736f;

typedef f32x4 f32x4_b4 __attribute__((aligned(4)));

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// ---------------------------------------------------------------------------
// Rows of a cache as MFMA operands.  A product over dims may take them in any
// order that both operands share, and so may the rows of a result, so each
// format has the order in which a lane's values are contiguous in memory.
//   key_dim:   dims 32 blk + ... of lane group a = lane / 16, j < 8
//   value_dim: dims 64 g + ... of lane m = lane % 16, j < 4
// ---------------------------------------------------------------------------
template <int FMT>
__device__ __forceinline__ uint32_t key_dim(uint32_t blk, uint32_t a, uint32_t j) {
    if (FMT == kKvQ4_0) return 32 * blk + 4 * a + (j & 3) + 16 * (j >> 2);
    return 32 * blk + 8 * a + j;
}
template <int FMT>
__device__ __forceinline__ uint32_t value_dim(uint32_t g, uint32_t m, uint32_t j) {
    if (FMT == kKvQ4_0) return 64 * g + 32 * (m >> 3) + 2 * (m & 7) + (j & 1) + 16 * (j >> 1);
    return 64 * g + 4 * m + j;
}

template <int FMT>
__device__ __forceinline__ uint64_t head_offset(uint32_t head, uint32_t head_dim) {
    if (FMT == kKvF32) return static_cast<uint64_t>(head) * head_dim * 4;
    return static_cast<uint64_t>(head) * (head_dim / 32) * (FMT == kKvQ8_0 ? 34 : 18);
}

typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef u32x2_t u32x2_a2 __attribute__((aligned(2)));

// The 8 values of block `blk` of a key row's head that lane group `a` holds.
template <int FMT>
__device__ __forceinline__ void load_key8(const uint8_t* head, uint32_t blk, uint32_t a, uint32_t head_dim, float* v) {
    if constexpr (FMT == kKvF32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t dim = 32 * blk + 8 * a + 4 * h;
            f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (dim < head_dim) x = *reinterpret_cast<const f32x4*>(head + dim * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * h + j] = x[j];
        }
    } else if (32 * blk >= head_dim) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    } else if constexpr (FMT == kKvQ8_0) {
        const uint8_t* p = head + blk * 34;
        const float d = h2f(*reinterpret_cast<const uint16_t*>(p));
        const u32x2_t c = *reinterpret_cast<const u32x2_a2*>(p + 2 + 8 * a);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = static_cast<float>(static_cast<int8_t>((j < 4 ? c.x : c.y) >> (8 * (j & 3)))) * d;
    } else {
        const uint8_t* p = head + blk * 18;
        const float d = h2f(*reinterpret_cast<const uint16_t*>(p));
        const uint32_t c = *reinterpret_cast<const u32_a2*>(p + 2 + 4 * a);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = static_cast<float>(static_cast<int>((c >> (8 * (j & 3) + 4 * (j >> 2))) & 15u) - 8) * d;
    }
}

// The 4 values of group `g` of a value row's head that lane m holds.
template <int FMT>
__device__ __forceinline__ void load_value4(const uint8_t* head, uint32_t g, uint32_t m, uint32_t head_dim, float* v) {
    const uint32_t dim = value_dim<FMT>(g, m, 0);
    if (dim >= head_dim) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = 0.0f;
    } else if constexpr (FMT == kKvF32) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(head + dim * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x[j];
    } else if constexpr (FMT == kKvQ8_0) {
        const uint8_t* p = head + (dim / 32) * 34;
        const float d = h2f(*reinterpret_cast<const uint16_t*>(p));
        const uint32_t c = *reinterpret_cast<const u32_a2*>(p + 2 + dim % 32);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = static_cast<float>(static_cast<int8_t>(c >> (8 * j))) * d;
    } else {
        const uint8_t* p = head + (dim / 32) * 18;
        const float d = h2f(*reinterpret_cast<const uint16_t*>(p));
        const uint32_t c = *reinterpret_cast<const uint16_t*>(p + 2 + 2 * (m & 7));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = static_cast<float>(static_cast<int>((c >> (8 * (j & 1) + 4 * (j >> 1))) & 15u) - 8) * d;
    }
}

struct AttnParams {
    const float* q;
    const uint8_t* prefix;       // K plane; V plane prefix_plane bytes on
    const uint8_t* cache;        // K plane; V plane cache_plane bytes on
    const uint32_t* lengths;
    float* partial_out;          // [slot][kv head][row][head_dim]
    float2* partial_ml;          // [slot][kv head][row]
    float* scores;               // [sequence][kv head][row][score_pitch], or null
    uint64_t prefix_plane, cache_plane;
    uint32_t row_bytes, prefix_length, capacity, score_pitch;
    uint32_t tokens, q_heads, kv_heads, group, head_dim;
    uint32_t rows;               // of one KV head: sequences * tokens * group
    uint32_t seq_rows;           // tokens * group
    uint32_t prefix_tiles, prefix_slots, own_tiles, own_slots, prefix_items;
    float scale;                 // with log2(e)
};

// The prompt by f16 pieces (prefix_attention_wide.hip), items = prefix_tiles *
// prefix_slots * kv_heads: 64 rows to a workgroup and tile, or 128 with the
// prompt packed into `room` (attn_packed_bytes) first.
hipError_t launch_attn_wide(hipStream_t stream, int format, uint32_t items, const AttnParams& a, void* room);
uint64_t attn_packed_bytes(uint32_t head_dim, uint32_t kv_heads, uint32_t prefix_length);

}  // namespace atlas
