// prefix_attention.hpp -- what the kernels of the shared-prompt attention have
// in common: how lanes read the rows of a cache, and a call's parameters.
#pragma once

#include "device_common.hpp"
#include "launch.hpp"

namespace atlas {

inline constexpr int kAttnThreads = 256;
inline constexpr int kAttnWaves = kAttnThreads / kWave;
inline constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// The maximum over lanes that differ in bit 3 / 4 / 5 of their number.
__device__ __forceinline__ float max_xor8(float x) { return fmaxf(x, dpp_f32<0x128, 0xf, false>(x)); }  // row_ror:8
__device__ __forceinline__ float max_xor16(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float max_xor32(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_xor16(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float sum_xor32(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// ---------------------------------------------------------------------------
// Rows of a cache as MFMA operands.  A product over dims may take them in any
// order that both operands share, and so may the rows of a result, so each
// format has the order in which a lane's values are contiguous in memory:
// units of 8 key dims and quads of 4 value dims.
// ---------------------------------------------------------------------------
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef u32x2_t u32x2_a2 __attribute__((aligned(2)));
typedef u32x4_t u32x4_a2 __attribute__((aligned(2)));

// The dims of unit 4 blk + a, j < 8.
template <int FMT>
__device__ __forceinline__ uint32_t key_dim(uint32_t blk, uint32_t a, uint32_t j) {
    if (FMT == kKvQ4_0) return 32 * blk + 4 * a + (j & 3) + 16 * (j >> 2);
    return 32 * blk + 8 * a + j;
}

template <int FMT>
__device__ __forceinline__ uint64_t head_offset(uint32_t head, uint32_t head_dim) {
    if (FMT == kKvF32) return static_cast<uint64_t>(head) * head_dim * 4;
    return static_cast<uint64_t>(head) * (head_dim / 32) * (FMT == kKvQ8_0 ? 34 : 18);
}

constexpr uint32_t kNowhere = 0x7ffffff0u;  // a buffer offset past every span: reads as zero

// The dims that value quad q (of head_dim / 4) holds, e < 4.
template <int FMT>
__device__ __forceinline__ uint32_t quad_dim(uint32_t q, uint32_t e) {
    if (FMT == kKvQ4_0) return 32 * (q >> 3) + 2 * (q & 7) + (e & 1) + 16 * (e >> 1);
    return 4 * q + e;
}

// The rows of a plane that a tile covers, from `first` on: `rows` of them are
// there (0: none, `first` is then some row that is).  f32 rows come through a
// buffer that ends with them: what a lane asks for past them, or past the head's
// dims (offset kNowhere), is zero.  Quantised rows lie on 2-byte boundaries, where
// buffer loads of more than 2 bytes have returned zeros inside the buffer: they
// come by plain loads, from the last row or the head's first block where there
// is nothing, and whoever unpacks them takes nothing of those.
template <int FMT>
struct TileRows;
template <>
struct TileRows<kKvF32> {
    __amdgpu_buffer_rsrc_t rs;
    uint32_t row_bytes;
    __device__ TileRows(const uint8_t* plane, uint32_t first, uint32_t rows, uint32_t row_bytes, uint32_t head_off)
        : rs(span_rsrc(plane + static_cast<uint64_t>(first) * row_bytes, rows ? rows * row_bytes - head_off : 0u)),
          row_bytes(row_bytes) {}
    __device__ f32x4 quad(uint32_t row, uint32_t off) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, row * row_bytes + off, 0, 0));
    }
};
struct QuantTileRows {
    const uint8_t* base;
    uint32_t row_bytes, rows;
    __device__ QuantTileRows(const uint8_t* plane, uint32_t first, uint32_t rows, uint32_t row_bytes)
        : base(plane + static_cast<uint64_t>(first) * row_bytes), row_bytes(row_bytes), rows(rows) {}
    // one 32-bit offset from a base that all lanes share
    template <typename T>
    __device__ T at(uint32_t row, uint32_t off, uint32_t behind) const {
        const uint32_t last = rows ? rows - 1 : 0u;
        return *reinterpret_cast<const T*>(base + (__umul24(min(row, last), row_bytes) + (off == kNowhere ? 0u : off) + behind));
    }
};
template <>
struct TileRows<kKvQ8_0> : QuantTileRows {
    __device__ TileRows(const uint8_t* plane, uint32_t first, uint32_t rows, uint32_t row_bytes, uint32_t)
        : QuantTileRows(plane, first, rows, row_bytes) {}
};
template <>
struct TileRows<kKvQ4_0> : QuantTileRows {
    __device__ TileRows(const uint8_t* plane, uint32_t first, uint32_t rows, uint32_t row_bytes, uint32_t)
        : QuantTileRows(plane, first, rows, row_bytes) {}
};

// The low four bits of byte i, less 8: bytes convert in one instruction.
__device__ __forceinline__ float nibble(uint32_t w, int i) {
    return static_cast<float>((w & 0x0f0f0f0fu) >> (8 * i) & 255u) - 8.0f;
}

// 8 key dims as stored (unit c = 4 blk + a, the dims of key_dim); offset is
// the first of them, for a quantised row its block's scale.  codes() leaves
// the stored numbers and returns what they are times: nothing where the key or
// the dims are not `there`.  That is asked here and not at the load, and the
// empty asm holds the unpacking here too: either, moved up behind the load,
// waits for it and leaves nothing in flight (64 rows x 100003 Q8_0 41 us).
template <int FMT>
struct RawKey;
template <>
struct RawKey<kKvF32> {
    f32x4 x[2];
    static __device__ uint32_t offset(uint32_t unit, uint32_t head_dim, uint32_t part) {
        const uint32_t dim = 8 * unit + 4 * part;
        return dim < head_dim ? dim * 4 : kNowhere;
    }
    __device__ void load(const TileRows<kKvF32>& t, uint32_t row, uint32_t, const uint32_t (&o)[2]) {
        x[0] = t.quad(row, o[0]);
        x[1] = t.quad(row, o[1]);
    }
    __device__ float codes(float (&v)[8], bool) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[j >> 2][j & 3];
        return 1.0f;
    }
};
template <>
struct RawKey<kKvQ8_0> {
    u32x2_t c;
    uint16_t d;
    static __device__ uint32_t offset(uint32_t unit, uint32_t head_dim, uint32_t) {
        return 8 * unit < head_dim ? (unit >> 2) * 34 : kNowhere;
    }
    __device__ void load(const TileRows<kKvQ8_0>& t, uint32_t row, uint32_t unit, const uint32_t (&o)[2]) {
        c = t.at<u32x2_a2>(row, o[0], 2 + 8 * (unit & 3));
        d = t.at<uint16_t>(row, o[0], 0);
    }
    __device__ float codes(float (&v)[8], bool there) const {
        uint32_t c0 = c.x, c1 = c.y, scale = d;
        asm volatile("" : "+v"(c0), "+v"(c1), "+v"(scale));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(static_cast<int8_t>((j < 4 ? c0 : c1) >> (8 * (j & 3))));
        return there ? h2f(static_cast<uint16_t>(scale)) : 0.0f;
    }
};
template <>
struct RawKey<kKvQ4_0> {
    uint32_t c;
    uint16_t d;
    static __device__ uint32_t offset(uint32_t unit, uint32_t head_dim, uint32_t) {
        return 8 * unit < head_dim ? (unit >> 2) * 18 : kNowhere;
    }
    __device__ void load(const TileRows<kKvQ4_0>& t, uint32_t row, uint32_t unit, const uint32_t (&o)[2]) {
        c = t.at<u32_a2>(row, o[0], 2 + 4 * (unit & 3));
        d = t.at<uint16_t>(row, o[0], 0);
    }
    __device__ float codes(float (&v)[8], bool there) const {
        uint32_t c0 = c, scale = d;
        asm volatile("" : "+v"(c0), "+v"(scale));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = nibble(j < 4 ? c0 : c0 >> 4, j & 3);
        return there ? h2f(static_cast<uint16_t>(scale)) : 0.0f;
    }
};
// 4 value dims as stored.
template <int FMT>
struct RawValue;
template <>
struct RawValue<kKvF32> {
    f32x4 x;
    static __device__ uint32_t offset(uint32_t quad, uint32_t head_dim) { return 4 * quad < head_dim ? quad * 16 : kNowhere; }
    __device__ void load(const TileRows<kKvF32>& t, uint32_t row, uint32_t, uint32_t o) { x = t.quad(row, o); }
    __device__ float codes(float (&v)[4], bool) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x[j];
        return 1.0f;
    }
};
template <>
struct RawValue<kKvQ8_0> {
    uint32_t c;
    uint16_t d;
    static __device__ uint32_t offset(uint32_t quad, uint32_t head_dim) {
        return 4 * quad < head_dim ? (quad >> 3) * 34 : kNowhere;
    }
    __device__ void load(const TileRows<kKvQ8_0>& t, uint32_t row, uint32_t quad, uint32_t o) {
        c = t.at<u32_a2>(row, o, 2 + 4 * (quad & 7));
        d = t.at<uint16_t>(row, o, 0);
    }
    __device__ float codes(float (&v)[4], bool there) const {
        uint32_t c0 = c, scale = d;
        asm volatile("" : "+v"(c0), "+v"(scale));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = static_cast<float>(static_cast<int8_t>(c0 >> (8 * j)));
        return there ? h2f(static_cast<uint16_t>(scale)) : 0.0f;
    }
};
template <>
struct RawValue<kKvQ4_0> {
    uint16_t c, d;
    static __device__ uint32_t offset(uint32_t quad, uint32_t head_dim) {
        return 4 * quad < head_dim ? (quad >> 3) * 18 : kNowhere;
    }
    __device__ void load(const TileRows<kKvQ4_0>& t, uint32_t row, uint32_t quad, uint32_t o) {
        c = t.at<uint16_t>(row, o, 2 + 2 * (quad & 7));
        d = t.at<uint16_t>(row, o, 0);
    }
    __device__ float codes(float (&v)[4], bool there) const {
        uint32_t c0 = c, scale = d;
        asm volatile("" : "+v"(c0), "+v"(scale));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = nibble(j < 2 ? c0 : c0 >> 4, j & 1);
        return there ? h2f(static_cast<uint16_t>(scale)) : 0.0f;
    }
};

// The numbers themselves: f32 holds a code times a block's scale exactly.
template <class Raw, int N>
__device__ __forceinline__ void raw_values(const Raw& raw, float (&v)[N], bool there) {
    const float s = raw.codes(v, there);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] *= s;
}

// The dims of unit `unit` of a query row, scaled.
template <int FMT>
__device__ __forceinline__ void load_query8(const float* q, uint32_t unit, uint32_t head_dim, float scale, float (&x)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t dim = key_dim<FMT>(unit / 4, unit % 4, 4 * h);
        const bool there = dim < head_dim;
        const f32x4 v = *reinterpret_cast<const f32x4*>(q + (there ? dim : 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * h + j] = there ? v[j] * scale : 0.0f;
    }
}

// The four values of quad q of a row in LDS.
template <int FMT>
__device__ __forceinline__ void put_quad(float* row, uint32_t q, f32x4 v) {
    if constexpr (FMT == kKvQ4_0) {
        *reinterpret_cast<f32x2_t*>(row + quad_dim<FMT>(q, 0)) = f32x2_t{v.x, v.y};
        *reinterpret_cast<f32x2_t*>(row + quad_dim<FMT>(q, 2)) = f32x2_t{v.z, v.w};
    } else {
        *reinterpret_cast<f32x4*>(row + 4 * q) = v;
    }
}

// Part `i` of `parts` of `rows` rows, in whole units of `unit`: no two parts
// differ by more than one.
__device__ __forceinline__ void part_of(uint32_t rows, uint32_t unit, uint32_t i, uint32_t parts, uint32_t& begin, uint32_t& end) {
    const uint32_t units = (rows + unit - 1) / unit, each = units / parts, more = units % parts;
    begin = min((i * each + min(i, more)) * unit, rows);
    end = min(begin + (each + (i < more ? 1u : 0u)) * unit, rows);
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
inline constexpr uint32_t kMostPromptKeys = 1u << 16;  // of a segment
hipError_t launch_attn_wide(hipStream_t stream, int format, uint32_t items, const AttnParams& a, void* room);
uint64_t attn_packed_bytes(uint32_t head_dim, uint32_t kv_heads, uint32_t prefix_length);

}  // namespace atlas
