// prefix_attention_wide.hip -- the prompt's segments of the shared-prompt
// attention when a batch has many query rows.  Reading the prompt's cache once
// leaves products: 4 head_dim operations per (row, key), which the f32 matrix
// instructions bound at 154 TFLOP/s.  Here every f32 operand is the sum of two
// f16, x = hi + lo, |x - hi - lo| <= 2^-22 |x|, and a product is three on the
// f16 matrix cores (hi hi + hi lo + lo hi; lo lo is below the rounding), summed
// in f32.
//
// f16 has five exponent bits, so operands are scaled by powers of two first,
// which loses nothing: each query row and each key row to its own largest
// magnitude in [2^14, 2^15) (the exponents are added back to the score), and
// each value row likewise, v' = v 2^{-ev}.  A weight 2^{x - m} (m about the
// row's largest x) takes its value row's exponent before it is split,
// p' = 2^{x - m} 2^{ev + m - m'} with m' about the row's largest x + ev, so
// that sum 2^x v = 2^{m'} sum p' v' keeps every row's precision whatever the
// rows' scales.  m and m' are whole numbers: all these factors are exact.
//
// A workgroup of four wavefronts takes 32 RW query rows and walks one segment
// in tiles of KT keys: the tile's rows come from the cache as they are stored,
// one tile ahead, and are converted once, into the fragments that the matrix
// instructions read (LDS, 16 bytes a lane, in lane order: no bank conflicts).
// A wavefront holds 32 rows' queries and accumulators in registers; S^T = K Q^T
// leaves a query row in a lane, so its maximum and sum are the lane's own, and
// P^T is the operand of O^T = V^T P^T without leaving its registers.
#include "prefix_attention.hpp"

namespace atlas {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

constexpr uint32_t kNowhere = 0x7ffffff0u;  // a buffer offset past every span: reads as zero

__device__ __forceinline__ float max_mag(float a, float b) { return fmaxf(__builtin_fabsf(a), __builtin_fabsf(b)); }

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
__device__ __forceinline__ float sum_xor32(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// The exponent e that brings a row of largest magnitude `top` to
// [2^14, 2^15) as x 2^-e; rows below 2^-low are taken as 2^-low.
__device__ __forceinline__ int row_exponent(float top, int low) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    return (e < -low ? -low : e) - 14;
}

// x 2^-e as two f16 vectors.
struct Pieces {
    half8 hi, lo;
};
__device__ __forceinline__ Pieces pieces(const float (&x)[8]) {
    Pieces p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2_t y = {x[2 * i], x[2 * i + 1]};
        const half2_t h = __builtin_convertvector(y, half2_t);
        const f32x2_t rest = {y.x - static_cast<float>(h.x), y.y - static_cast<float>(h.y)};
        const half2_t l = __builtin_convertvector(rest, half2_t);
        p.hi[2 * i] = h.x;
        p.hi[2 * i + 1] = h.y;
        p.lo[2 * i] = l.x;
        p.lo[2 * i + 1] = l.y;
    }
    return p;
}

// The dims that value quad q (of head_dim / 4) holds, e < 4.
template <int FMT>
__device__ __forceinline__ uint32_t quad_dim(uint32_t q, uint32_t e) {
    if (FMT == kKvQ4_0) return 32 * (q >> 3) + 2 * (q & 7) + (e & 1) + 16 * (e >> 1);
    return 4 * q + e;
}

// Raw bytes of 8 key dims (unit c = 4 blk + a, the dims of key_dim) and of 4
// value dims, through a buffer whose end is the last key's: what lies past it
// is zero.
template <int FMT>
struct RawKey;
template <>
struct RawKey<kKvF32> {
    f32x4 x[2];
    static __device__ uint32_t offset(uint32_t unit, uint32_t head_dim, uint32_t part) {
        const uint32_t dim = 8 * unit + 4 * part;
        return dim < head_dim ? dim * 4 : kNowhere;
    }
    __device__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row, const uint32_t (&o)[2]) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
            x[p] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, row + o[p], 0, 0));
    }
    __device__ void values(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[j >> 2][j & 3];
    }
};
template <>
struct RawKey<kKvQ8_0> {
    u32x2_t c;
    uint16_t d;
    static __device__ uint32_t offset(uint32_t unit, uint32_t head_dim, uint32_t part) {
        if (8 * unit >= head_dim) return kNowhere;
        return (unit >> 2) * 34 + (part ? 0 : 2 + 8 * (unit & 3));
    }
    __device__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row, const uint32_t (&o)[2]) {
        c = __builtin_amdgcn_raw_buffer_load_b64(rs, row + o[0], 0, 0);
        d = __builtin_amdgcn_raw_buffer_load_b16(rs, row + o[1], 0, 0);
    }
    __device__ void values(float (&v)[8]) const {
        const float s = h2f(d);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(static_cast<int8_t>((j < 4 ? c.x : c.y) >> (8 * (j & 3)))) * s;
    }
};
template <>
struct RawKey<kKvQ4_0> {
    uint32_t c;
    uint16_t d;
    static __device__ uint32_t offset(uint32_t unit, uint32_t head_dim, uint32_t part) {
        if (8 * unit >= head_dim) return kNowhere;
        return (unit >> 2) * 18 + (part ? 0 : 2 + 4 * (unit & 3));
    }
    __device__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row, const uint32_t (&o)[2]) {
        c = __builtin_amdgcn_raw_buffer_load_b32(rs, row + o[0], 0, 0);
        d = __builtin_amdgcn_raw_buffer_load_b16(rs, row + o[1], 0, 0);
    }
    __device__ void values(float (&v)[8]) const {
        const float s = h2f(d);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(static_cast<int>((c >> (8 * (j & 3) + 4 * (j >> 2))) & 15u) - 8) * s;
    }
};
template <int FMT>
struct RawValue;
template <>
struct RawValue<kKvF32> {
    f32x4 x;
    static __device__ uint32_t offset(uint32_t quad, uint32_t head_dim, uint32_t part) {
        return 4 * quad < head_dim ? quad * 16 : kNowhere;
    }
    __device__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row, const uint32_t (&o)[2]) {
        x = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, row + o[0], 0, 0));
    }
    __device__ void values(float (&v)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x[j];
    }
};
template <>
struct RawValue<kKvQ8_0> {
    uint32_t c;
    uint16_t d;
    static __device__ uint32_t offset(uint32_t quad, uint32_t head_dim, uint32_t part) {
        if (4 * quad >= head_dim) return kNowhere;
        return (quad >> 3) * 34 + (part ? 0 : 2 + 4 * (quad & 7));
    }
    __device__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row, const uint32_t (&o)[2]) {
        c = __builtin_amdgcn_raw_buffer_load_b32(rs, row + o[0], 0, 0);
        d = __builtin_amdgcn_raw_buffer_load_b16(rs, row + o[1], 0, 0);
    }
    __device__ void values(float (&v)[4]) const {
        const float s = h2f(d);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = static_cast<float>(static_cast<int8_t>(c >> (8 * j))) * s;
    }
};
template <>
struct RawValue<kKvQ4_0> {
    uint16_t c, d;
    static __device__ uint32_t offset(uint32_t quad, uint32_t head_dim, uint32_t part) {
        if (4 * quad >= head_dim) return kNowhere;
        return (quad >> 3) * 18 + (part ? 0 : 2 + 2 * (quad & 7));
    }
    __device__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row, const uint32_t (&o)[2]) {
        c = __builtin_amdgcn_raw_buffer_load_b16(rs, row + o[0], 0, 0);
        d = __builtin_amdgcn_raw_buffer_load_b16(rs, row + o[1], 0, 0);
    }
    __device__ void values(float (&v)[4]) const {
        const float s = h2f(d);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = static_cast<float>((c >> (8 * (j & 1) + 4 * (j >> 1)) & 15) - 8) * s;
    }
};

// Sizes of a kernel: D the head_dim it is padded to, RW row tiles of 32.
template <int D, int RW>
struct Wide {
    static constexpr int KW = kAttnWaves / RW;                  // wavefronts that share a row tile
    static constexpr int KT = (RW == 4 ? 32 : 64) * 256 / D;    // keys of a tile
    static constexpr int MT = KT / KW / 32;                     // of which a wavefront takes MT blocks of 32
    static constexpr int KS = D / 16;                           // steps of a score
    static constexpr int DT = D / 32;                           // blocks of an output row
    static constexpr int BUFS = RW == 4 ? 2 : 1;
    static constexpr int kKeyFrags = KT / 32 * KS * 2;          // of 1 KiB
    static constexpr int kValueFrags = KT / 32 * DT * 2 * 2;
    static constexpr int KI = KT / 32;                          // keys a lane converts
    static constexpr int KU = D / 64;                           // units of each
    static constexpr int VI = KT * D / 8192;                    // value groups a lane converts
};

template <int D, int RW>
struct WideTile {
    half8 key[Wide<D, RW>::kKeyFrags][kWave];
    half8 value[Wide<D, RW>::kValueFrags][kWave];
    int key_exp[Wide<D, RW>::KT];        // of the key row
    int value_exp[Wide<D, RW>::KT];      // of the value row, also as a float
    float value_expf[Wide<D, RW>::KT];
    float value_scale[Wide<D, RW>::KT];  // 2^-value_exp
};

template <int FMT, int D, int RW>
struct WideRaw {
    RawKey<FMT> key[Wide<D, RW>::KI][Wide<D, RW>::KU];
    RawValue<FMT> value[Wide<D, RW>::VI][8];
};

// Where this lane's part of a tile lies.
template <int FMT, int D, int RW>
struct WideLane {
    uint32_t key_off[Wide<D, RW>::KU][2], value_off[2];
    uint32_t key_row, value_row;  // first key of each; the others a constant on
    static constexpr uint32_t kQuads = D / 4;
    __device__ WideLane(uint32_t lane, uint32_t wave, uint32_t head_dim) {
#pragma unroll
        for (int u = 0; u < Wide<D, RW>::KU; ++u)
#pragma unroll
            for (uint32_t p = 0; p < 2; ++p) key_off[u][p] = RawKey<FMT>::offset(lane / 8 + 8 * u, head_dim, p);
        key_row = 8 * wave + lane % 8;
        // value groups of 8 keys: kWave / kQuads to a wavefront
        const uint32_t group = wave * (kWave / kQuads) + lane / kQuads;
        value_row = 32 * (group / 4) + 16 * (group / 2 % 2) + 4 * (group % 2);
#pragma unroll
        for (uint32_t p = 0; p < 2; ++p) value_off[p] = RawValue<FMT>::offset(lane % kQuads, head_dim, p);
    }
};

template <int FMT, int D, int RW>
__device__ __forceinline__ void load_tile(WideRaw<FMT, D, RW>& raw, const WideLane<FMT, D, RW>& at, const uint8_t* keys,
                                          const uint8_t* values, uint32_t first, uint32_t end, uint32_t row_bytes,
                                          uint32_t head_off) {
    using W = Wide<D, RW>;
    const uint32_t rows = first < end ? min(end - first, static_cast<uint32_t>(W::KT)) : 0u;
    const uint32_t bytes = rows ? rows * row_bytes - head_off : 0u;
    const uint64_t base = static_cast<uint64_t>(first) * row_bytes;
    const __amdgpu_buffer_rsrc_t k = span_rsrc(keys + base, bytes), v = span_rsrc(values + base, bytes);
#pragma unroll
    for (int i = 0; i < W::KI; ++i)
#pragma unroll
        for (int u = 0; u < W::KU; ++u) raw.key[i][u].load(k, (at.key_row + 32 * i) * row_bytes, at.key_off[u]);
#pragma unroll
    for (int i = 0; i < W::VI; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            raw.value[i][j].load(v, (at.value_row + i * (kAttnWaves * (256 / D) * 8) + 8 * (j >> 2) + (j & 3)) * row_bytes,
                                 at.value_off);
}

template <int FMT, int D, int RW>
__device__ __forceinline__ void convert_keys(const WideRaw<FMT, D, RW>& raw, WideTile<D, RW>& tile, uint32_t lane,
                                             uint32_t wave) {
    using W = Wide<D, RW>;
#pragma unroll
    for (int i = 0; i < W::KI; ++i) {
        float x[W::KU][8];
        float top = 0.0f;
#pragma unroll
        for (int u = 0; u < W::KU; ++u) {
            raw.key[i][u].values(x[u]);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max_mag(top, x[u][j]);
        }
        top = max_xor32(max_xor16(max_xor8(top)));
        const int e = row_exponent(top, 100);
        const float scale = pow2i(-e);
        const uint32_t key = 32 * i + 8 * wave + lane % 8;
        if (lane < 8) tile.key_exp[key] = e;
#pragma unroll
        for (int u = 0; u < W::KU; ++u) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[u][j] *= scale;
            const Pieces p = pieces(x[u]);
            const uint32_t unit = lane / 8 + 8 * u;
            const uint32_t frag = (i * W::KS + unit / 2) * 2, to = unit % 2 * 32 + (8 * wave + lane % 8);
            tile.key[frag][to] = p.hi;
            tile.key[frag + 1][to] = p.lo;
        }
    }
}

template <int FMT, int D, int RW>
__device__ __forceinline__ void convert_values(const WideRaw<FMT, D, RW>& raw, WideTile<D, RW>& tile, uint32_t lane,
                                               uint32_t wave) {
    using W = Wide<D, RW>;
    constexpr uint32_t kQuads = D / 4;
#pragma unroll
    for (int i = 0; i < W::VI; ++i) {
        const uint32_t group = (wave + kAttnWaves * i) * (kWave / kQuads) + lane / kQuads, quad = lane % kQuads;
        const uint32_t key0 = 32 * (group / 4) + 16 * (group / 2 % 2) + 4 * (group % 2);
        float x[8][4];  // [key][dim]
        float top[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            raw.value[i][j].values(x[j]);
            top[j] = fmaxf(max_mag(x[j][0], x[j][1]), max_mag(x[j][2], x[j][3]));
        }
        // eight maxima over the group's lanes: each step halves what a lane
        // keeps, ending with key lane % 8
        float t4[4], t2[2];
        const bool b2 = lane & 4, b1 = lane & 2, b0 = lane & 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) t4[j] = fmaxf(b2 ? top[4 + j] : top[j], dpp_f32<0x141, 0xf, false>(b2 ? top[j] : top[4 + j]));
#pragma unroll
        for (int j = 0; j < 2; ++j) t2[j] = fmaxf(b1 ? t4[2 + j] : t4[j], dpp_f32<0x1b, 0xf, false>(b1 ? t4[j] : t4[2 + j]));
        float m = fmaxf(b0 ? t2[1] : t2[0], dpp_f32<0xb1, 0xf, false>(b0 ? t2[0] : t2[1]));
        m = max_xor8(m);
        if (kQuads >= 32) m = max_xor16(m);
        if (kQuads >= 64) m = max_xor32(m);
        if (quad < 8) {
            const uint32_t key = key0 + 8 * (quad / 4) + quad % 4;
            const int e = row_exponent(m, 76);
            tile.value_exp[key] = e;
            tile.value_expf[key] = static_cast<float>(e);
            tile.value_scale[key] = pow2i(-e);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const f32x4 s0 = *reinterpret_cast<const f32x4*>(&tile.value_scale[key0]);
        const f32x4 s1 = *reinterpret_cast<const f32x4*>(&tile.value_scale[key0 + 8]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = x[j][e] * (j < 4 ? s0[j & 3] : s1[j & 3]);
            const Pieces p = pieces(y);
            // block and row of dim e of the quad: consecutive quads are
            // consecutive lanes of one block
            const uint32_t block = D == 64 ? e / 2 : 4 * (quad / 32) + e;
            const uint32_t m_row = D == 64 ? quad + 16 * (e % 2) : quad % 32;
            const uint32_t frag = (((group / 4) * W::DT + block) * 2 + group / 2 % 2) * 2;
            const uint32_t to = 32 * (group % 2) + m_row;
            tile.value[frag][to] = p.hi;
            tile.value[frag + 1][to] = p.lo;
        }
    }
}

// The dim that row m of output block dt holds.
template <int FMT, int D>
__device__ __forceinline__ uint32_t output_dim(uint32_t dt, uint32_t m) {
    if (D == 64) return quad_dim<FMT>(m % 16, 2 * dt + m / 16);
    return quad_dim<FMT>(32 * (dt / 4) + m, dt % 4);
}

template <int FMT, int D, int RW>
__global__ __launch_bounds__(kAttnThreads, 1) void attn_wide_kernel(AttnParams a) {
    using W = Wide<D, RW>;
    __shared__ WideTile<D, RW> tiles[W::BUFS];
    const uint32_t lane = threadIdx.x % kWave, n = lane % 32, side = lane / 32;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    const uint32_t row_wave = wave % RW, key_wave = wave / RW;

    // workgroups of one segment on one XCD, whose L2 then reads it once
    uint32_t item = blockIdx.x, slot, tile_index, kv_head;
    if (a.prefix_slots % 8 == 0) {
        const uint32_t xcd = item % 8;
        item /= 8;
        tile_index = item % a.prefix_tiles;
        item /= a.prefix_tiles;
        slot = item % (a.prefix_slots / 8) * 8 + xcd;
        kv_head = item / (a.prefix_slots / 8);
    } else {
        tile_index = item % a.prefix_tiles;
        item /= a.prefix_tiles;
        slot = item % a.prefix_slots;
        kv_head = item / a.prefix_slots;
    }
    const uint32_t part = ((a.prefix_length + a.prefix_slots - 1) / a.prefix_slots + W::KT - 1) / W::KT * W::KT;
    const uint32_t begin = min(slot * part, a.prefix_length), end = min(begin + part, a.prefix_length);
    const uint32_t head_off = static_cast<uint32_t>(head_offset<FMT>(kv_head, a.head_dim));
    const uint8_t* keys = a.prefix + head_off;
    const uint8_t* values = a.prefix + a.prefix_plane + head_off;

    // 32 query rows as operands: lane (row n, side) holds the dims of unit 2 s + side
    const uint32_t row = tile_index * 32 * RW + row_wave * 32 + n;
    const uint32_t at = min(row, a.rows - 1);
    const float* q_row =
        a.q + (static_cast<uint64_t>(at / a.group) * a.q_heads + kv_head * a.group + at % a.group) * a.head_dim;
    half8 q_hi[W::KS], q_lo[W::KS];
    int q_exp;
    {
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < W::KS; ++s) {
            const uint32_t unit = 2 * s + side;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t dim = key_dim<FMT>(unit / 4, unit % 4, j);
                top = max_mag(top, dim < a.head_dim ? q_row[dim] * a.scale : 0.0f);
            }
        }
        top = max_xor32(top);
        q_exp = row_exponent(top, 100);
        const float scale = pow2i(-q_exp);
#pragma unroll
        for (int s = 0; s < W::KS; ++s) {
            const uint32_t unit = 2 * s + side;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t dim = key_dim<FMT>(unit / 4, unit % 4, j);
                x[j] = dim < a.head_dim ? q_row[dim] * a.scale * scale : 0.0f;
            }
            const Pieces p = pieces(x);
            q_hi[s] = p.hi;
            q_lo[s] = p.lo;
        }
    }

    const WideLane<FMT, D, RW> mine(lane, wave, a.head_dim);
    WideRaw<FMT, D, RW> raw;
    f32x16 out[W::DT];
#pragma unroll
    for (int d = 0; d < W::DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) out[d][i] = 0.0f;
    // whole numbers; every x <= m + 8 and x + ev <= mv + 8, so a weight
    // 2^(x - m) is at most 2^8 and p' = 2^(x + ev - mv + 6) at most 2^14
    float m = neg_inf(), mv = neg_inf(), l = 0.0f;

    load_tile(raw, mine, keys, values, begin, end, a.row_bytes, head_off);
    if (W::BUFS == 2) {
        convert_keys(raw, tiles[0], lane, wave);
        convert_values(raw, tiles[0], lane, wave);
        load_tile(raw, mine, keys, values, begin + W::KT, end, a.row_bytes, head_off);
        __syncthreads();
    }
    int buf = 0;
    for (uint32_t first = begin; first < end; first += W::KT) {
        if (W::BUFS == 2) {
            convert_keys(raw, tiles[buf ^ 1], lane, wave);
            convert_values(raw, tiles[buf ^ 1], lane, wave);
            load_tile(raw, mine, keys, values, first + 2 * W::KT, end, a.row_bytes, head_off);
        } else {
            convert_keys(raw, tiles[0], lane, wave);
            convert_values(raw, tiles[0], lane, wave);
            load_tile(raw, mine, keys, values, first + W::KT, end, a.row_bytes, head_off);
            __syncthreads();
        }
        const uint32_t left = end - first;
        const WideTile<D, RW>& tile = tiles[W::BUFS == 2 ? buf : 0];
#pragma unroll
        for (int mt = 0; mt < W::MT; ++mt) {
            const uint32_t block = key_wave * W::MT + mt;
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < W::KS; ++k) {
                const half8 hi = tile.key[(block * W::KS + k) * 2][lane], lo = tile.key[(block * W::KS + k) * 2 + 1][lane];
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo, q_hi[k], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, q_lo[k], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, q_hi[k], s, 0, 0, 0);
            }
            // register i: key 8 (i / 4) + 4 side + i % 4 of the block
            typedef int i32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const i32x4 e = *reinterpret_cast<const i32x4*>(&tile.key_exp[32 * block + 8 * g + 4 * side]);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * g + j] = __builtin_ldexpf(s[4 * g + j], e[j] + q_exp);
            }
            if (left < W::KT) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * block + 8 * (i / 4) + 4 * side + i % 4 >= left) s[i] = neg_inf();
            }
            float top = neg_inf(), top_v = neg_inf();
            i32x4 ev[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t key = 32 * block + 8 * g + 4 * side;
                const f32x4 e = *reinterpret_cast<const f32x4*>(&tile.value_expf[key]);
                ev[g] = *reinterpret_cast<const i32x4*>(&tile.value_exp[key]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    top = fmaxf(top, s[4 * g + j]);
                    top_v = fmaxf(top_v, s[4 * g + j] + e[j]);
                }
            }
            top = max_xor32(top);
            top_v = max_xor32(top_v);
            if (__builtin_amdgcn_ballot_w64(top > m + 8.0f || top_v > mv + 8.0f) != 0) {
                const float m_new = fmaxf(m, __builtin_ceilf(top)), mv_new = fmaxf(mv, __builtin_ceilf(top_v));
                l *= m == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
                const float fade = mv == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(mv - mv_new);
                m = m_new;
                mv = mv_new;
#pragma unroll
                for (int d = 0; d < W::DT; ++d) out[d] *= fade;
            }
            const float base = m == neg_inf() ? 0.0f : m;
            const int shift = m == neg_inf() ? 0 : static_cast<int>(m - mv) + 6;
            half8 p_hi[2], p_lo[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float w = __builtin_amdgcn_exp2f(s[8 * h + j] - base);
                    l += w;
                    p[j] = __builtin_ldexpf(w, ev[2 * h + j / 4][j % 4] + shift);
                }
                const Pieces x = pieces(p);
                p_hi[h] = x.hi;
                p_lo[h] = x.lo;
            }
#pragma unroll
            for (int d = 0; d < W::DT; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t frag = ((block * W::DT + d) * 2 + h) * 2;
                    const half8 hi = tile.value[frag][lane], lo = tile.value[frag + 1][lane];
                    out[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo, p_hi[h], out[d], 0, 0, 0);
                    out[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, p_lo[h], out[d], 0, 0, 0);
                    out[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, p_hi[h], out[d], 0, 0, 0);
                }
        }
        __syncthreads();
        buf ^= 1;
    }

    // out relative to 2^m, as l is
    l = sum_xor32(l);
    const int back = m == neg_inf() ? 0 : static_cast<int>(mv - m) - 6;
#pragma unroll
    for (int d = 0; d < W::DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) out[d][i] = __builtin_ldexpf(out[d][i], back);
    if constexpr (W::KW == 2) {
        // the second wavefront of a row tile hands its sums over through LDS
        float* room = reinterpret_cast<float*>(&tiles[0]) + row_wave * (32 * (D + 2));
        if (key_wave == 1) {
            if (side == 0) {
                room[32 * D + n] = m;
                room[32 * D + 32 + n] = l;
            }
#pragma unroll
            for (int d = 0; d < W::DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) room[(d * 16 + i) * kWave + lane] = out[d][i];
        }
        __syncthreads();
        if (key_wave == 1) return;
        const float m2 = room[32 * D + n], l2 = room[32 * D + 32 + n];
        const float both = fmaxf(m, m2);
        const float f1 = m == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(m - both);
        const float f2 = m2 == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(m2 - both);
        m = both;
        l = l * f1 + l2 * f2;
#pragma unroll
        for (int d = 0; d < W::DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) out[d][i] = out[d][i] * f1 + room[(d * 16 + i) * kWave + lane] * f2;
    }
    if (row >= a.rows) return;
    const uint64_t to = (static_cast<uint64_t>(slot) * a.kv_heads + kv_head) * a.rows + row;
    if (side == 0) a.partial_ml[to] = make_float2(m, l);
    float* p = a.partial_out + to * a.head_dim;
#pragma unroll
    for (int d = 0; d < W::DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t dim = output_dim<FMT, D>(d, 8 * (i / 4) + 4 * side + i % 4);
            if (dim < a.head_dim) p[dim] = out[d][i];
        }
}

template <int FMT, int D>
void launch_wide(hipStream_t stream, uint32_t items, uint32_t row_waves, const AttnParams& a) {
    if (row_waves == 4)
        hipLaunchKernelGGL((attn_wide_kernel<FMT, D, 4>), dim3(items), dim3(kAttnThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((attn_wide_kernel<FMT, D, 2>), dim3(items), dim3(kAttnThreads), 0, stream, a);
}

template <int FMT>
void launch_wide(hipStream_t stream, uint32_t items, uint32_t row_waves, const AttnParams& a) {
    if (a.head_dim <= 64)
        launch_wide<FMT, 64>(stream, items, row_waves, a);
    else if (a.head_dim <= 128)
        launch_wide<FMT, 128>(stream, items, row_waves, a);
    else
        launch_wide<FMT, 256>(stream, items, row_waves, a);
}

}  // namespace

hipError_t launch_attn_wide(hipStream_t stream, int format, uint32_t items, uint32_t row_waves, const AttnParams& a) {
    if (format == kKvF32)
        launch_wide<kKvF32>(stream, items, row_waves, a);
    else if (format == kKvQ8_0)
        launch_wide<kKvQ8_0>(stream, items, row_waves, a);
    else
        launch_wide<kKvQ4_0>(stream, items, row_waves, a);
    return hipGetLastError();
}

}  // namespace atlas
