// paged_attention.hpp -- attention of one new token of each sequence over the
// sequence's pages (paged_layout.hpp), for the translation units of its formats.
//
// For query head h of sequence b, with KV head h / group:
//   x_j = scale * (q . k_j) over positions lo <= j < length whose page is there,
//         lo = max(0, length - window), or 0 without a window,
//   out = sum_j e^{x_j} v_j / sum_j e^{x_j}, zero where nothing is seen.
// One pass over the keys with the running maximum and sum.  The work is split
// evenly, not row by row: a row is a sequence's KV head with up to 16 query
// heads, its positions are counted in units of a wavefront's step, and of all
// rows' units together every workgroup takes the same number, so that lengths do
// not matter for the balance and a lone sequence keeps the whole chip.  Lengths
// live on the device, so the workgroups find their parts there.  A part that ends
// inside a row leaves its maximum m, sum l of 2^{x - m} and sum O of 2^{x - m} v,
// which a second launch joins.  (Short rows are not cut: whole_row_units.)
//
// Bound by its loads and, behind which they do not wholly hide, a step's chain of
// products and conversions: 24 sequences of 1000 to 30001 Q8_0 positions, 8 KV heads of
// 128 dims and 32 heads 173 to 176 us, 4.6 TB/s (the loads alone 5.8); 131072 f16
// positions of 256 dims 34 us with the join, 4.0 TB/s.  Q4_0 is bound by its unpacking: 261001
// positions of 256 dims 28 us, 940 vector instructions of a wavefront for 32 positions.
#pragma once

#include "attention_lanes.hpp"
#include "paged_plan.hpp"

namespace atlas {

struct PagedAttnParams {
    const float* q;
    const uint8_t* pages;
    const uint32_t* table;
    const uint32_t* lengths;
    float* output;
    float* partial_out;   // [2 parts][heads][head_dim]
    float2* partial_ml;   // [2 parts][heads]
    PagedRow* rows;       // [sequences][kv_heads][head_tiles], of rows that see something
    uint64_t page_bytes;
    uint32_t part_bytes, page_count, page_shift, table_width, sequences, capacity;
    uint32_t kv_heads, group, head_tiles, heads, q_heads, head_dim, window;
    // the join's last argument, in the second line of them: a third one costs it 0.3 us
    uint32_t most_parts, few_parts, part_units;  // parts of all work; units of a part where there are more than few_parts
    float scale;                                 // with log2(e)
    uint32_t row_units;                          // rows are not split, and have as many units at most; 0: they are
};

// The positions that a sequence's token sees, and their units.
struct SeenRange {
    uint32_t lo, hi;
};
__device__ __forceinline__ SeenRange seen_of(const PagedAttnParams& a, uint32_t seq) {
    const uint32_t length = min(a.lengths[seq], a.capacity);
    return {a.window && length > a.window ? length - a.window : 0u, length};
}
__device__ __forceinline__ uint32_t units_of(SeenRange s, uint32_t unit) {
    return s.hi > s.lo ? (s.hi + unit - 1) / unit - s.lo / unit : 0u;
}
// Of at most 2^30 units, and one more for a row whose window begins and ends inside units.
__device__ __forceinline__ uint32_t parts_of(const PagedAttnParams& a, uint32_t total) {
    uint32_t parts = (total + a.part_units - 1) / a.part_units;
    parts = parts > a.few_parts ? parts : a.few_parts;
    parts = parts < a.most_parts ? parts : a.most_parts;
    return parts < total ? parts : total;
}

__device__ __forceinline__ uint32_t uniform_u32(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(v)); }

constexpr uint32_t kPastPage = 0x7ffffff0u;  // a buffer offset past every part: reads as zero

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ u32x4_t load16(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t base) {
    return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, off, base, 0));
}
__device__ __forceinline__ u32x2_t load8(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t base) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(rs, off, base, 0));
}
__device__ __forceinline__ uint32_t load4(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t base) {
    return __builtin_amdgcn_raw_buffer_load_b32(rs, off, base, 0);
}

// A head's rows of one page, from row `row` on: 16 keys.  A page that is not
// there has no bytes, and every load of it is zero.
struct PageRows {
    __amdgpu_buffer_rsrc_t keys, values;
    uint32_t row;
    __device__ PageRows(const PagedAttnParams& a, uint32_t kv_head, uint32_t page, uint32_t row)
        : keys(span_rsrc(base(a, page, kv_head), page < a.page_count ? a.part_bytes : 0u)),
          values(span_rsrc(base(a, page, a.kv_heads + kv_head), page < a.page_count ? a.part_bytes : 0u)), row(row) {}
    static __device__ const uint8_t* base(const PagedAttnParams& a, uint32_t page, uint32_t part) {
        return a.pages + (page < a.page_count ? page : 0u) * a.page_bytes + static_cast<uint64_t>(part) * a.part_bytes;
    }
};

// Blocks of a value row in runs of 8, 4, 2, 1 (paged_run), and the 32-bit words
// in which a lane holds its codes: BLOCK bytes of each block.
template <int NB, int BLOCK>
struct ValueWords {
    uint8_t first[NB] = {}, run[NB] = {}, word[NB] = {};
    int words = 0;
    constexpr ValueWords() {
        int b = 0;
        for (int r = 8; r; r /= 2)
            if (NB & r) {
                for (int i = 0; i < r; ++i) {
                    first[b + i] = static_cast<uint8_t>(b);
                    run[b + i] = static_cast<uint8_t>(r);
                    word[b + i] = static_cast<uint8_t>(words);
                }
                words += r * BLOCK < 4 ? 1 : r * BLOCK / 4;
                b += r;
            }
    }
};

// What a wavefront holds of its step's keys and values, lane c + 16 g: of a tile
// of 16 keys, key c's dims of group g; of the values, 16 lanes' dims of the keys
// 4 g + r.  Scores come out as S^T = K Q^T: lane (c, g) has the scores of head c
// with keys 4 g + r of each tile, which is the operand that O^T = V^T P^T wants if
// the order of its keys is (tile, r) for each g; so P never leaves its lane and
// a head's statistics are the lane's own.
template <int FMT, int NB, int HP>
struct Step;

// f32 throughout (v_mfma_f32_16x16x4): at the 151 TFLOP/s of a large product 19 TB/s
// of keys and values, whatever the number of heads.
template <int NB>
struct Step<kKvF32, NB, 16> {
    static constexpr int kTiles = 1, kOut = 2 * NB, kQuads = NB / 2, kQueryBytes = 2 * NB * kWave * 16;
    static constexpr float kUnscale = 1.0f;
    f32x4 k[2 * NB];
    f32x4 v[4][kQuads ? kQuads : 1];
    f32x2_t v2[4];
    __device__ __forceinline__ void load_keys(const PageRows (&p)[1], uint32_t c, uint32_t g, uint32_t head_dim) {
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
            const uint32_t dim = 16 * s + 4 * g;
            const uint32_t off = s < 2 * NB - 2 || dim < head_dim ? c * head_dim * 4 + dim * 4 : kPastPage;
            k[s] = __builtin_bit_cast(f32x4, load16(p[0].keys, off, p[0].row * head_dim * 4));
        }
    }
    __device__ __forceinline__ void load_values(const PageRows (&p)[1], uint32_t c, uint32_t g, uint32_t head_dim) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t line = (4 * g + r) * head_dim * 4;
#pragma unroll
            for (int u = 0; u < kQuads; ++u) {
                const uint32_t dim = 64 * u + 4 * c;
                v[r][u] = __builtin_bit_cast(f32x4, load16(p[0].values, dim < head_dim ? line + dim * 4 : kPastPage, p[0].row * head_dim * 4));
            }
            if constexpr (NB % 2) {
                const uint32_t dim = 64 * kQuads + 2 * c;
                v2[r] = __builtin_bit_cast(f32x2_t, load8(p[0].values, dim < head_dim ? line + dim * 4 : kPastPage, p[0].row * head_dim * 4));
            }
        }
    }
    static __device__ __forceinline__ uint32_t query_lane(uint32_t c, uint32_t g) { return (c + 16 * g) * 16; }
    __device__ __forceinline__ void scores(const uint8_t* queries, uint32_t, float, f32x4 (&s)[1]) const {
        f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
        s[0] = t;
#pragma unroll
        for (int i = 0; i < 2 * NB; i += 2) {
            const f32x4 q0 = *reinterpret_cast<const f32x4*>(queries + i * 1024), q1 = *reinterpret_cast<const f32x4*>(queries + i * 1024 + 1024);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i][j], q0[j], s[0], 0, 0, 0);
                t = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i + 1][j], q1[j], t, 0, 0, 0);
            }
            if (i % 4) __builtin_amdgcn_sched_barrier(0);
        }
        s[0] += t;
    }
    // values of keys that are not seen must not be numbers that are none
    __device__ __forceinline__ void keep(const bool (&seen)[1][4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int u = 0; u < kQuads; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[r][u][j] = seen[0][r] ? v[r][u][j] : 0.0f;
            if constexpr (NB % 2) v2[r] = f32x2_t{seen[0][r] ? v2[r].x : 0.0f, seen[0][r] ? v2[r].y : 0.0f};
        }
    }
    __device__ __forceinline__ void add(const f32x4 (&p)[1], f32x4 (&out)[kOut]) const {
        // one rounding of the long sums for the step's keys, not one for every four
#pragma unroll
        for (int u = 0; u < kQuads; ++u) {
            f32x4 sum[4] = {};
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][u][j], p[0][r], sum[j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[4 * u + j] += sum[j];
        }
        if constexpr (NB % 2) {
            f32x4 sum[2] = {};
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < 2; ++j) sum[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v2[r][j], p[0][r], sum[j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 2; ++j) out[4 * kQuads + j] += sum[j];
        }
    }
    // O^T has dims in its rows: tile 4 u + j row i is dim 64 u + 4 i + j
    static __device__ __forceinline__ void put(float* line, uint32_t, uint32_t g, const f32x4 (&out)[kOut]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int u = 0; u < kQuads; ++u)
                *reinterpret_cast<f32x4*>(line + 64 * u + 16 * g + 4 * r) =
                    f32x4{out[4 * u][r], out[4 * u + 1][r], out[4 * u + 2][r], out[4 * u + 3][r]};
            if constexpr (NB % 2)
                *reinterpret_cast<f32x2_t*>(line + 64 * kQuads + 8 * g + 2 * r) = f32x2_t{out[4 * kQuads][r], out[4 * kQuads + 1][r]};
        }
    }
    static __device__ constexpr uint32_t query_dim(uint32_t j) { return j; }
};

// Two f16 numbers that add up to x, each rounded to nearest: 2^-24 of x at most is
// lost, or 2^-25 where the second one is below 2^-14.
__device__ __forceinline__ void f16_pieces(float x, _Float16& hi, _Float16& lo) {
    hi = static_cast<_Float16>(materialize(x));
    lo = static_cast<_Float16>(materialize(x - static_cast<float>(hi)));
}

// Products of f16 (v_mfma_f32_16x16x32_f16): keys and values as they are, the
// other factor as two f16 numbers, brought near f16's largest by a power of two
// that the sums are divided by.  A query's pieces lose 2^-24 of each number, or
// 2^-39 of the row's largest; a weight's 2^-24, or 2^-40.  (A product lines its terms up by
// their operands' exponents, 2^-14 for all f16 numbers below it: of a weight of 2^15 such a
// value loses what is below 2^-23, of a query's largest number such a key 2^-37.)  A value's load has 16 bytes a
// lane: the address unit takes 17 cycles for any of whole rows (65 for a key's), and
// twice the loads of 8 took 32.2 us for 30.2 (256 windows of 512 of 256 dims).
template <int NB>
struct Step<kKvF16, NB, 16> {
    static constexpr int kTiles = 2, kOut = 2 * NB, kEights = NB / 4, kFours = NB % 4 / 2, kQueryBytes = 2 * NB * kWave * 16;
    static constexpr float kUnscale = 0x1p-15f;
    static constexpr uint32_t kItemsPadded = 4 * NB;
    u32x4_t k[2][NB];
    u32x4_t v[8][kEights ? kEights : 1];  // eight dims a lane of runs of 128, then four of one of 64, two of one of 32
    u32x2_t v4[8];
    uint32_t v2[8];
    __device__ __forceinline__ void load_keys(const PageRows (&p)[2], uint32_t c, uint32_t g, uint32_t head_dim) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < NB; ++s) {
                const uint32_t dim = 32 * s + 8 * g;
                const uint32_t off = s < NB - 1 || dim < head_dim ? (c * head_dim + dim) * 2 : kPastPage;
                k[h][s] = load16(p[h].keys, off, p[h].row * head_dim * 2);
            }
    }
    __device__ __forceinline__ void load_values(const PageRows (&p)[2], uint32_t c, uint32_t g, uint32_t head_dim) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const PageRows& rows = p[j / 4];
            const uint32_t line = (4 * g + j % 4) * head_dim * 2;
#pragma unroll
            for (int u = 0; u < kEights; ++u) {
                const uint32_t dim = 128 * u + 8 * c;
                v[j][u] = load16(rows.values, dim < head_dim ? line + dim * 2 : kPastPage, rows.row * head_dim * 2);
            }
            if constexpr (kFours) {
                const uint32_t dim = 128 * kEights + 4 * c;
                v4[j] = load8(rows.values, dim < head_dim ? line + dim * 2 : kPastPage, rows.row * head_dim * 2);
            }
            if constexpr (NB % 2) {
                const uint32_t dim = 32 * (NB - 1) + 2 * c;
                v2[j] = load4(rows.values, dim < head_dim ? line + dim * 2 : kPastPage, rows.row * head_dim * 2);
            }
        }
    }
    static __device__ __forceinline__ uint32_t query_lane(uint32_t c, uint32_t g) { return (c + 16 * g) * 16; }
    static __device__ __forceinline__ void put_query(uint8_t* room, uint32_t head, uint32_t it, f16x8_t hi, f16x8_t lo) {
        uint8_t* to = room + it / 4 * 2048 + (it % 4 * 16 + head) * 16;
        *reinterpret_cast<f16x8_t*>(to) = hi;
        *reinterpret_cast<f16x8_t*>(to + 1024) = lo;
    }
    __device__ __forceinline__ void scores(const uint8_t* queries, uint32_t, float unscale, f32x4 (&s)[2]) const {
        s[0] = s[1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const f16x8_t hi = *reinterpret_cast<const f16x8_t*>(queries + b * 2048);
            const f16x8_t lo = *reinterpret_cast<const f16x8_t*>(queries + b * 2048 + 1024);
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k[h][b]), hi, s[h], 0, 0, 0);
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k[h][b]), lo, s[h], 0, 0, 0);
            if (b % 2) __builtin_amdgcn_sched_barrier(0);
        }
        s[0] *= unscale;
        s[1] *= unscale;
    }
    __device__ __forceinline__ void keep(const bool (&seen)[2][4]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t mask = seen[j / 4][j % 4] ? 0xffffffffu : 0u;
#pragma unroll
            for (int u = 0; u < kEights; ++u) v[j][u] &= mask;
            if constexpr (kFours) v4[j] &= mask;
            if constexpr (NB % 2) v2[j] &= mask;
        }
    }
    // dims 2 pair + e of eight keys
    template <int E>
    static __device__ __forceinline__ f16x8_t column(const uint32_t (&w)[8]) {
        u32x4_t x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], E ? 0x07060302u : 0x05040100u);
        return __builtin_bit_cast(f16x8_t, x);
    }
    __device__ __forceinline__ void add(const f32x4 (&p)[2], f32x4 (&out)[kOut]) const {
        f16x8_t hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            _Float16 a, b;
            f16_pieces(p[j / 4][j % 4] * 0x1p15f, a, b);
            hi[j] = a;
            lo[j] = b;
        }
        const auto one = [&](f16x8_t x, f32x4& o) {
            f32x4 sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, hi, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
            sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, lo, sum, 0, 0, 0);
            o += sum;
        };
#pragma unroll
        for (int i = 0; i < NB; ++i) {  // the words that a lane holds of a row
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[j] = i < 4 * kEights ? v[j][i / 4 % (kEights ? kEights : 1)][i % 4] : i < 4 * kEights + 2 * kFours ? v4[j][i % 2] : v2[j];
            one(column<0>(w), out[2 * i]);
            one(column<1>(w), out[2 * i + 1]);
        }
    }
    // O^T has dims in its rows: tile 2 i + e row k is dim 2 i + e of the lane's run k
    static __device__ __forceinline__ void put(float* line, uint32_t, uint32_t g, const f32x4 (&out)[kOut]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t k = 4 * g + r;
#pragma unroll
            for (int i = 0; i < 4 * kEights; i += 2)
                *reinterpret_cast<f32x4*>(line + i / 4 * 128 + 8 * k + i % 4 * 2) = f32x4{out[2 * i][r], out[2 * i + 1][r], out[2 * i + 2][r], out[2 * i + 3][r]};
            if constexpr (kFours) {
                constexpr int i = 4 * kEights;
                *reinterpret_cast<f32x4*>(line + 32 * i + 4 * k) = f32x4{out[2 * i][r], out[2 * i + 1][r], out[2 * i + 2][r], out[2 * i + 3][r]};
            }
            if constexpr (NB % 2) *reinterpret_cast<f32x2_t*>(line + 32 * (NB - 1) + 2 * k) = f32x2_t{out[2 * NB - 2][r], out[2 * NB - 1][r]};
        }
    }
    static __device__ constexpr uint32_t query_dim(uint32_t j) { return j; }
};

// Products of codes, which f16 and bf16 hold as they are, with two f16 numbers for
// a query's (as above) and, for the weights times the values' scales, three bf16
// numbers: the 24 bits of an f32, cut in three, over its whole range.  A key's
// scale goes on the product of its block, a value's on the weight, so codes are
// only unpacked.
//
// A lane loads 16 bytes of a key at once: loads of 8 or 4 bytes a lane, rows apart,
// keep the address unit busy for 64 cycles whatever they bring (4.7 and 2.4 TB/s of
// the 6.2 that 16 bytes reach).  They are another block than its neighbours'.  So
// lanes exchange words until a product has one block's dims, whose scale goes on the
// result; or, of Q8_0's two blocks and 8 heads at most, each column takes one (its
// query is zero for the other's), with twice the products and half the scales (256
// dims, 8 heads: 88 us for 95; Q4_0 the other way, 71 for 77).  A product has 16
// columns and a row HP heads at most (4, 8 or 16): for the keys columns are (piece of
// the query or block, head), for the values (block, head), so that a lane cuts the
// weights of one block in 16 / HP, not of all.
template <int FMT, int NB, int HP>
struct Step {
    static_assert(FMT == kKvQ8_0 || FMT == kKvQ4_0);
    static constexpr bool kBytes = FMT == kKvQ8_0;
    static constexpr int kTiles = 2, kOut = 2 * NB, kBlock = kBytes ? 2 : 1, kRow = NB * (kBytes ? 32 : 16);
    static constexpr ValueWords<NB, kBlock> kWords{};
    // v_cvt_off_f32_i4 gives sixteenths
    static constexpr float kUnscale = kBytes ? 1.0f : 16.0f;
    // keys: blocks of the 64 bytes that lanes g load at once, and of a product; products that the query's pieces make;
    // in LDS a query's 64 lanes for each product
    static constexpr int kKeyBlocks = kBytes ? 2 : 4, kKeySteps = (NB + kKeyBlocks - 1) / kKeyBlocks;
    static constexpr bool kExchanged = !kBytes || HP == 16;
    static constexpr int kSpan = kExchanged ? 1 : 2, kSpans = (NB + kSpan - 1) / kSpan, kPieces = kExchanged && HP < 16 ? 1 : 2;
    // values: blocks to the columns
    static constexpr int kValueBlocks = 16 / HP, kValueSteps = (NB + kValueBlocks - 1) / kValueBlocks;
    static constexpr int kQueryBytes = kSpans * kSpan * kPieces * 1024;
    static constexpr uint32_t kItemsPadded = 4 * kSpans * kSpan;

    u32x4_t k[2][kKeySteps];
    u32x2_t ks[2][kSpans], vs[2][kValueSteps];  // scales of keys 4 g + r
    uint32_t v[8][kWords.words];

    static __device__ __forceinline__ uint32_t query_lane(uint32_t c, uint32_t g) { return (c + 16 * g) * 16; }
    // Item `it` of a head's query, 8 dims of block it / 4, for the lane that has their codes.
    static __device__ __forceinline__ void put_query(uint8_t* room, uint32_t head, uint32_t it, f16x8_t hi, f16x8_t lo) {
        const uint32_t block = it / 4, quarter = it % 4;
        f16x8_t* to = reinterpret_cast<f16x8_t*>(room);
        if constexpr (kExchanged) {
            to += block * kPieces * 64 + (kBytes ? quarter % 2 * 2 + quarter / 2 : quarter) * 16 + head;
            *to = HP < 16 && head / HP % 2 ? lo : hi;
            if constexpr (HP == 16) to[64] = lo;
        } else if (head < 8) {
            to += (block % kSpans * 2 + quarter % 2) * 128 + (block / kSpans * 2 + quarter / 2) * 16 + head;
            const uint32_t mine = block / kSpans * 8, others = 8 - mine;
            to[mine] = hi;
            to[mine + 64] = lo;
            to[others] = to[others + 64] = f16x8_t{};
        }
    }
    // Of a lane's blocks, one behind the other, two at a time.  Behind a row's blocks lie other rows', or nothing: the
    // columns that take those are no block's, and no one reads them.
    template <int BLOCKS>
    static __device__ __forceinline__ void load_scales(__amdgpu_buffer_rsrc_t rs, uint32_t page_shift, uint32_t row, uint32_t g,
                                                       uint32_t block, u32x2_t (&s)[BLOCKS]) {
        const uint32_t base = (kRow << page_shift) + row / 4 * NB * 8, off = (g * NB + block) * 8;
#pragma unroll
        for (int i = 0; i + 1 < BLOCKS; i += 2) {
            const u32x4_t x = load16(rs, off + 8 * i, base);
            s[i] = u32x2_t{x[0], x[1]};
            s[i + 1] = u32x2_t{x[2], x[3]};
        }
        if constexpr (BLOCKS % 2) s[BLOCKS - 1] = load8(rs, off + 8 * (BLOCKS - 1), base);
    }
    __device__ __forceinline__ void load_keys(const PageRows (&p)[2], uint32_t c, uint32_t g, uint32_t page_shift) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < kKeySteps; ++i) {
                const uint32_t in_row = kExchanged ? i * 64 + 16 * g : (g / 2 * kSpans + i) * 32 + g % 2 * 16;
                const uint32_t off = (kExchanged ? (i + 1) * 64 <= kRow : NB % 2 == 0) || in_row < kRow ? c * kRow + in_row : kPastPage;
                k[h][i] = load16(p[h].keys, off, p[h].row * kRow);
            }
            load_scales(p[h].keys, page_shift, p[h].row, g, kExchanged ? 0 : c / 8 * kSpans, ks[h]);
        }
    }
    __device__ __forceinline__ void load_values(const PageRows (&p)[2], uint32_t c, uint32_t g, uint32_t page_shift) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __amdgpu_buffer_rsrc_t rs = p[j / 4].values;
            const uint32_t base = p[j / 4].row * kRow, line = (4 * g + j % 4) * kRow;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (kWords.first[b] != b) continue;  // a run starts here
                const int bytes = kWords.run[b] * kBlock, w = kWords.word[b];
                const uint32_t off = line + 16 * kBlock * b + c * bytes;
                if (bytes == 16) {
                    const u32x4_t x = load16(rs, off, base);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[j][(w + i) % kWords.words] = x[i];
                } else if (bytes == 8) {
                    const u32x2_t x = load8(rs, off, base);
#pragma unroll
                    for (int i = 0; i < 2; ++i) v[j][(w + i) % kWords.words] = x[i];
                } else if (bytes == 4) {
                    v[j][w] = load4(rs, off, base);
                } else if (bytes == 2) {
                    v[j][w] = static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(rs, off, base, 0));
                } else {
                    v[j][w] = static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(rs, off, base, 0));
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) load_scales(p[h].values, page_shift, p[h].row, g, c / HP * kValueSteps, vs[h]);
    }
    // Eight codes of a key as f16: 1024 + (a code without its sign) has it in its low
    // bits, or 16 times it four bits higher up.  Written out where the compiler makes
    // two instructions of one.
    static __device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
        uint32_t y;
        asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(y) : "v"(x), "s"(mask), "v"(bits));
        return y;
    }
    static __device__ __forceinline__ f16x8_t key_codes(u32x2_t w) {
        u32x4_t x;
        const auto less = [](uint32_t y, float by) {
            const f16x2_t z = {static_cast<_Float16>(by), static_cast<_Float16>(by)};
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, y) - z);
        };
        if constexpr (kBytes) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = less(__builtin_amdgcn_perm(0x64646464u, w[i / 2] ^ 0x80808080u, i % 2 ? 0x04030402u : 0x04010400u), 1152.0f);
        } else {
            const f16x2_t sixteenth = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
            const f16x2_t minus72 = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const uint32_t y = i ? w[0] >> 8 : w[0];
                x[i] = less(and_or(y, 0x000f000fu, 0x64006400u), 1032.0f);
                // (1024 + 16 n) / 16 - 72 = n - 8
                x[i + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, and_or(y, 0x00f000f0u, 0x64006400u)),
                                                                                  sixteenth, minus72));
            }
        }
        return __builtin_bit_cast(f16x8_t, x);
    }
    static __device__ __forceinline__ float scale_of(u32x2_t s, int r) { return h2f(static_cast<uint16_t>(s[r / 2] >> (16 * (r % 2)))); }
    // Words i, j of lanes g and of lanes g ^ 2 or g ^ 1 change places where they are off the diagonal.
    static __device__ __forceinline__ void exchange32(u32x4_t& w, int i, int j) {
        const auto p = __builtin_amdgcn_permlane32_swap(w[i], w[j], false, false);
        w[i] = p[0];
        w[j] = p[1];
    }
    static __device__ __forceinline__ void exchange16(u32x4_t& w, int i, int j) {
        const auto p = __builtin_amdgcn_permlane16_swap(w[i], w[j], false, false);
        w[i] = p[0];
        w[j] = p[1];
    }
    // From a lane's 16 bytes of one block its eight dims of each: of Q4_0's block b in word b, the dims of word g; of
    // Q8_0's in words 2 b and 2 b + 1, those of the half g % 2, quarter g / 2.
    static __device__ __forceinline__ u32x4_t exchange(u32x4_t w) {
        exchange32(w, 0, 2);
        exchange32(w, 1, 3);
        if constexpr (!kBytes) {
            exchange16(w, 0, 1);
            exchange16(w, 2, 3);
        }
        return w;
    }
    __device__ __forceinline__ void scores(const uint8_t* queries, uint32_t c, float unscale, f32x4 (&s)[2]) const {
        s[0] = s[1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kKeySteps; ++i) {
            const u32x4_t w[2] = {kExchanged ? exchange(k[0][i]) : k[0][i], kExchanged ? exchange(k[1][i]) : k[1][i]};
#pragma unroll
            for (int j = 0; j < kKeyBlocks / kSpan; ++j) {
                const int b = i * kKeyBlocks / kSpan + j;
                if (b >= kSpans) break;
                f32x4 d[2] = {};
#pragma unroll
                for (int m = 0; m < kSpan; ++m) {
                    f16x8_t x[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        x[h] = key_codes(kBytes ? u32x2_t{w[h][2 * (j + m) % 4], w[h][(2 * (j + m) + 1) % 4]} : u32x2_t{w[h][j], 0});
#pragma unroll
                    for (int n = 0; n < kPieces; ++n) {
                        const f16x8_t q = *reinterpret_cast<const f16x8_t*>(queries + ((b * kSpan + m) * kPieces + n) * 1024);
#pragma unroll
                        for (int h = 0; h < 2; ++h) d[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[h], q, d[h], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
                {
                    u32x2_t scale = ks[h][b];
                    if (kSpan == 2 && NB % 2 && b == kSpans - 1 && c >= 8) scale = u32x2_t{0, 0};  // no block's
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[h][r] = __builtin_fmaf(d[h][r], scale_of(scale, r), s[h][r]);
                }
                if (kSpan == 2 || j % 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the sums of a head's columns; every lane has its own head, c % HP
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (HP == 8 || !kExchanged) s[h][r] += dpp_f32<0x128, 0xf, false>(s[h][r]);  // row_ror:8
                else if constexpr (HP == 4) s[h][r] += dpp_f32<0x124, 0xf, false>(s[h][r]);            // row_ror:4
                s[h][r] *= unscale;
            }
    }
    __device__ __forceinline__ void keep(const bool (&seen)[2][4]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t mask = (seen[h][2 * i] ? 0xffffu : 0u) | (seen[h][2 * i + 1] ? 0xffff0000u : 0u);
#pragma unroll
                for (int b = 0; b < kValueSteps; ++b) vs[h][b][i] &= mask;
            }
    }
    static __device__ __forceinline__ uint32_t upper(float odd, float even) {  // their upper halves
        return __builtin_amdgcn_perm(__float_as_uint(odd), __float_as_uint(even), 0x07060302u);
    }
    static __device__ __forceinline__ float cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
    // The low four bits of byte i, in one instruction.
    static __device__ __forceinline__ float nibble(uint32_t w, int i) {
        float x;
        if (i == 0)
            asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(x) : "v"(w));
        else if (i == 1)
            asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(x) : "v"(w));
        else if (i == 2)
            asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(x) : "v"(w));
        else
            asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(x) : "v"(w));
        return x;
    }
    // code e of block b of eight keys
    __device__ __forceinline__ bf16x8_t value_codes(int b, int e) const {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int at = (b - kWords.first[b]) * kBlock + (kBytes ? e : 0);
            const uint32_t w = v[j][kWords.word[b] + at / 4];
            if constexpr (kBytes)
                x[j] = static_cast<float>(static_cast<int8_t>(w >> (8 * (at % 4))));
            else
                x[j] = nibble(e ? w >> 4 : w, at % 4);
        }
        u32x4_t y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = upper(x[2 * i + 1], x[2 * i]);
        return __builtin_bit_cast(bf16x8_t, y);
    }
    __device__ __forceinline__ void add(const f32x4 (&p)[2], f32x4 (&out)[kOut]) {
        if constexpr (!kBytes) {  // two's complement by the flip of bit 3, here for both codes of a byte
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < kWords.words; ++i) {
                    v[j][i] ^= 0x88888888u;
                    asm("" : "+v"(v[j][i]));
                }
        }
#pragma unroll
        for (int step = 0; step < kValueSteps; ++step) {
            u32x4_t piece[3];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float w[2];
#pragma unroll
                for (int j = 0; j < 2; ++j)  // a multiply-add takes the f16 scale as it is
                    w[j] = __builtin_fmaf(p[i / 2][i % 2 * 2 + j], scale_of(vs[i / 2][step], i % 2 * 2 + j), 0.0f);
#pragma unroll
                for (int n = 0; n < 3; ++n) {
                    piece[n][i] = upper(w[1], w[0]);
                    if (n == 2) break;
                    w[0] -= cut(w[0]);
                    w[1] -= cut(w[1]);
                }
            }
            // columns of other blocks hold what no one reads
#pragma unroll
            for (int b = step; b < NB; b += kValueSteps)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bf16x8_t x = value_codes(b, e);
                    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int n = 0; n < 3; ++n)
                        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8_t, piece[n]), sum, 0, 0, 0);
                    out[2 * b + e] += sum;
                }
        }
    }
    // tile 2 b + e row i is dim 32 b + 2 i + e
    static __device__ __forceinline__ void put(float* line, uint32_t c, uint32_t g, const f32x4 (&out)[kOut]) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (c / HP == b / kValueSteps)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    *reinterpret_cast<f32x2_t*>(line + 32 * b + 8 * g + 2 * r) = f32x2_t{out[2 * b][r], out[2 * b + 1][r]};
    }
    // the order in which key_codes gives a lane's eight dims
    static __device__ constexpr uint32_t query_dim(uint32_t j) { return kBytes ? j : j / 2 + j % 2 * 4; }
};

// A workgroup a part of the work, or a whole row: then no other sequence's length
// is asked for and nothing is left to join.
template <int FMT, int NB, int HP, int WAVES, bool WHOLE>
__global__ __launch_bounds__(WAVES * kWave, WAVES == 4 ? paged_occupancy(32 * NB) : (WAVES + 3) / 4) void paged_attention_kernel(PagedAttnParams a) {
    using S = Step<FMT, NB, HP>;
    constexpr uint32_t kThreads = WAVES * kWave;
    constexpr int kTiles = S::kTiles;
    constexpr bool kQuantised = FMT == kKvQ8_0 || FMT == kKvQ4_0;
    constexpr uint32_t kKeys = paged_keys(FMT), kDims = 32 * NB, kPitch = kDims + 4;
    static_assert(kKeys == 16 * kTiles);
    // queries in the products' order; at the end the wavefronts' sums
    __shared__ union Room {
        uint8_t queries[S::kQueryBytes];
        float sums[WAVES][HP][kPitch];
    } room;
    __shared__ float2 room_ml[WAVES][HP];
    __shared__ float room_unscale[kPagedHeads];
    __shared__ uint32_t room_units[WAVES];
    __shared__ uint32_t found_before, found_seq;
    const uint32_t lane = threadIdx.x % kWave, c = lane % 16, g = lane / 16;
    const uint32_t wave = uniform_u32(threadIdx.x / kWave);
    const uint32_t rows = a.kv_heads * a.head_tiles;  // of a sequence

    uint32_t begin, end, before = 0, seq, units, each = 0, longer = 0;
    SeenRange seen;
    if constexpr (WHOLE) {
        seq = blockIdx.x / rows;
        seen = seen_of(a, seq);
        units = uniform_u32(units_of(seen, kKeys));
        begin = blockIdx.x % rows * units;
        end = begin + units;
        if (units == 0) {
            const uint32_t row = blockIdx.x % rows, head0 = row % a.head_tiles * kPagedHeads;
            const uint32_t heads = min(a.group - head0, static_cast<uint32_t>(HP));
            float* to = a.output + (static_cast<uint64_t>(seq) * a.q_heads + row / a.head_tiles * a.group + head0) * a.head_dim;
            for (uint32_t i = threadIdx.x; i < heads * a.head_dim; i += kThreads) to[i] = 0.0f;
            return;
        }
    } else {
        // this workgroup's units of all sequences', and the sequence that the first lies in; parts have `each` units,
        // the first `longer` one more
        const auto share = [&](uint32_t all_units) {
            const uint32_t total = uniform_u32(all_units) * rows, parts = uniform_u32(parts_of(a, total));
            if (blockIdx.x >= parts) return false;
            each = uniform_u32(total / parts);
            longer = total - each * parts;
            begin = blockIdx.x * each + min(blockIdx.x, longer);
            end = begin + each + (blockIdx.x < longer ? 1 : 0);
            return true;
        };
        if (a.sequences <= kWave) {  // each wavefront for itself: one sequence 9.7 -> 9.0 us with the shares' 32 bits
            SeenRange of_lane = {0, 0};
            if (lane < a.sequences) of_lane = seen_of(a, lane);
            const uint32_t own = units_of(of_lane, kKeys), upto = wave_inclusive_scan_u32(own);
            if (!share(readlane_u32(upto, kWave - 1))) return;
            const uint32_t wanted = uniform_u32(begin / rows), from = upto - own;
            seq = static_cast<uint32_t>(__builtin_ctzll(__builtin_amdgcn_ballot_w64(wanted >= from && wanted - from < own)));
            before = readlane_u32(from, seq) * rows;
            seen = {readlane_u32(of_lane.lo, seq), readlane_u32(of_lane.hi, seq)};
            units = readlane_u32(own, seq);
        } else {
            // a chunk of sequences, one a thread: units up to each
            const auto scan = [&](uint32_t units, uint32_t& chunk) {
                uint32_t upto = wave_inclusive_scan_u32(units);
                __syncthreads();
                if (lane == kWave - 1) room_units[wave] = upto;
                __syncthreads();
                chunk = 0;
#pragma unroll
                for (uint32_t w = 0; w < WAVES; ++w) {
                    if (w == wave) upto += chunk;
                    chunk += room_units[w];
                }
                return upto;
            };
            uint32_t mine = 0, first_units = 0;
            for (uint32_t b = threadIdx.x; b < a.sequences; b += kThreads) {
                const uint32_t own = units_of(seen_of(a, b), kKeys);
                if (b < kThreads) first_units = own;
                mine += own;
            }
            uint32_t all_units;
            uint32_t upto = scan(mine, all_units);
            if (!share(all_units)) return;
            const uint32_t wanted = uniform_u32(begin / rows);
            uint32_t ahead = 0;
            for (uint32_t first = 0; first < a.sequences; first += kThreads) {
                const uint32_t b = first + threadIdx.x;
                uint32_t own = first_units, chunk = all_units;
                if (a.sequences > kThreads) {
                    if (first) own = b < a.sequences ? units_of(seen_of(a, b), kKeys) : 0u;
                    upto = scan(own, chunk);
                }
                const uint32_t from = ahead + upto - own;
                if (wanted >= from && wanted - from < own) {
                    found_before = from;
                    found_seq = b;
                }
                ahead += chunk;
                if (ahead > wanted) break;
            }
            __syncthreads();
            before = uniform_u32(found_before) * rows;
            seq = uniform_u32(found_seq);
            seen = seen_of(a, seq);
            units = uniform_u32(units_of(seen, kKeys));
        }
    }

    for (uint32_t at = begin; at < end;) {
        // a segment: units [t0, t1) of a row's `units`
        while (at >= before + units * rows) {
            before += units * rows;
            ++seq;
            seen = seen_of(a, seq);
            units = uniform_u32(units_of(seen, kKeys));
        }
        seen.lo = uniform_u32(seen.lo);
        seen.hi = uniform_u32(seen.hi);
        const uint32_t row = uniform_u32((at - before) / units);
        const uint32_t t0 = at - before - row * units, t1 = min(units, t0 + (end - at));
        if (!WHOLE && t0 == 0 && threadIdx.x == 0) {
            const uint32_t last = at + units - 1, short_from = longer * (each + 1);  // the row's last unit
            a.rows[seq * rows + row] = {blockIdx.x, last < short_from ? last / (each + 1) : longer + (last - short_from) / each};
        }
        at += t1 - t0;
        const uint32_t kv_head = row / a.head_tiles, head0 = row % a.head_tiles * kPagedHeads;
        const uint32_t heads = min(a.group - head0, static_cast<uint32_t>(HP));
        const uint64_t line0 = static_cast<uint64_t>(seq) * a.q_heads + kv_head * a.group + head0;

        // Unit t's keys start at (seen.lo / kKeys + t) * kKeys; the wavefronts take units in turn.
        const uint32_t* table = a.table + static_cast<uint64_t>(seq) * a.table_width;
        const uint32_t start = seen.lo / kKeys * kKeys, tw = t0 + wave;
        constexpr uint32_t kAhead = kWave / kTiles;  // units whose pages a wavefront's lanes hold
        uint32_t pages = 0, pages_from = tw;
        const auto look_up = [&](uint32_t t) {
            pages_from = t;
            const uint32_t entry = (start + (t + lane / kTiles * WAVES) * kKeys + lane % kTiles * 16) >> a.page_shift;
            pages = entry < a.table_width ? table[entry] : 0xffffffffu;
            // waited for here, and not by whoever reads it: that wait would be for every load of every step
            asm volatile("" : "+v"(pages));
        };
        S step;
        uint32_t page[kTiles];  // of the step that is loaded
        const auto load = [&](uint32_t t, bool keys) {
            const uint32_t key = start + t * kKeys, mask = (1u << a.page_shift) - 1;
            if constexpr (kTiles == 1) {
                const PageRows p[1] = {PageRows(a, kv_head, page[0], key & mask)};
                if (keys)
                    step.load_keys(p, c, g, a.head_dim);
                else
                    step.load_values(p, c, g, a.head_dim);
            } else {
                const PageRows p[2] = {PageRows(a, kv_head, page[0], key & mask), PageRows(a, kv_head, page[1], (key + 16) & mask)};
                const uint32_t size = kQuantised ? a.page_shift : a.head_dim;
                if (keys)
                    step.load_keys(p, c, g, size);
                else
                    step.load_values(p, c, g, size);
            }
        };
        // the pages of unit t; none where nothing is seen, which loads nothing
        const auto turn = [&](uint32_t t) {
            if (t < t1 && t - pages_from >= kAhead * WAVES) look_up(t);
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i) {
                const uint32_t key = start + t * kKeys + 16 * i;
                const bool some = t < t1 && key < seen.hi && key + 16 > seen.lo;
                page[i] = some ? readlane_u32(pages, (t - pages_from) / WAVES * kTiles + i) : 0xffffffffu;
            }
        };
        // the query's loads, the step's behind them, and then what is done with the query
        const uint32_t head = threadIdx.x / 16 % 16, sub = threadIdx.x % 16, real = head % HP;  // by the first four wavefronts
        constexpr int kEach = FMT == kKvF32 ? 4 : 8, kItems = (kDims / kEach + 15) / 16;
        f32x4 x[kItems][kEach / 4];
        {
            const float* q = a.q + (line0 + min(real, heads - 1)) * a.head_dim;
#pragma unroll
            for (int i = 0; i < kItems; ++i)
#pragma unroll
                for (int h = 0; h < kEach / 4; ++h) {
                    const uint32_t dim = (sub + 16 * i) * kEach + 4 * h;
                    x[i][h] = *reinterpret_cast<const f32x4*>(q + (dim < a.head_dim ? dim : 0));
                }
        }
        look_up(tw);
        turn(tw);
        load(tw, true);
        load(tw, false);
        __syncthreads();  // the last segment's sums have been read
        if (WAVES == 4 || wave < 4) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < kItems; ++i)
#pragma unroll
                for (int h = 0; h < kEach / 4; ++h) {
                    const bool there = (sub + 16 * i) * kEach + 4 * h < a.head_dim && real < heads;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[i][h][j] = there ? x[i][h][j] * a.scale : 0.0f;
                        top = fmaxf(top, __builtin_fabsf(x[i][h][j]));
                    }
                }
            if constexpr (FMT == kKvF32) {
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    const uint32_t item = sub + 16 * i;
                    if (item < kDims / 4) *reinterpret_cast<f32x4*>(room.queries + item / 4 * 1024 + (item % 4 * 16 + head) * 16) = x[i][0];
                }
            } else {
                top = fmaxf(top, dpp_f32<0xb1, 0xf, false>(top));
                top = fmaxf(top, dpp_f32<0x4e, 0xf, false>(top));
                top = fmaxf(top, dpp_f32<0x141, 0xf, false>(top));
                top = fmaxf(top, dpp_f32<0x140, 0xf, false>(top));
                // the row's largest to 2^13 .. 2^14
                int up = 0;
                if (top > 0.0f && top < __builtin_inff()) up = min(14 - __builtin_amdgcn_frexp_expf(top), 126);
                const float by = pow2i(up);
                if (sub == 0) room_unscale[head] = pow2i(-up);
                constexpr uint32_t kLast = S::kItemsPadded;
#pragma unroll
                for (int i = 0; i < static_cast<int>((kLast + 15) / 16); ++i) {
                    const uint32_t item = sub + 16 * i;
                    f16x8_t hi, lo;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        _Float16 p = static_cast<_Float16>(0.0f), r = p;
                        const uint32_t d = S::query_dim(j);
                        if (i < kItems) f16_pieces(x[i < kItems ? i : 0][d / 4][d % 4] * by, p, r);
                        hi[j] = p;
                        lo[j] = r;
                    }
                    if (item < kLast) S::put_query(room.queries, head, item, hi, lo);
                }
            }
        }
        __syncthreads();
        const float unscale = FMT == kKvF32 ? 1.0f : room_unscale[c % HP];
        const uint8_t* queries = room.queries + S::query_lane(c, g);

        float m = neg_inf(), l = 0.0f;
        f32x4 out[S::kOut];
#pragma unroll
        for (int i = 0; i < S::kOut; ++i) out[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t t = tw; t < t1; t += WAVES) {
            const uint32_t key0 = start + t * kKeys;
            bool there[kTiles], whole = key0 >= seen.lo && key0 + kKeys <= seen.hi;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                there[i] = page[i] < a.page_count;
                whole = whole && there[i];
            }
            f32x4 s[kTiles];
            step.scores(queries, c, unscale, s);
            turn(t + WAVES);
            load(t + WAVES, true);
            __builtin_amdgcn_sched_barrier(0);
            if (!whole) {
                bool sees[kTiles][4];
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t key = key0 + 16 * i + 4 * g + r;
                        sees[i][r] = there[i] && key >= seen.lo && key < seen.hi;
                        s[i][r] = sees[i][r] ? s[i][r] : neg_inf();
                    }
                step.keep(sees);
            }
            float top = neg_inf();
#pragma unroll
            for (int i = 0; i < kTiles; ++i) top = fmaxf(top, fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
            top = max_xor32(max_xor16(top));
            if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
                const float m_new = fmaxf(m, top);
                const float fade = m == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                l *= fade;
#pragma unroll
                for (int i = 0; i < S::kOut; ++i) out[i] *= fade;
            }
            const float base = m == neg_inf() ? 0.0f : m;
            float sum[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][r] = __builtin_amdgcn_exp2f(s[i][r] - base);
                sum[i] = (s[i][0] + s[i][1]) + (s[i][2] + s[i][3]);
            }
            l += kTiles == 1 ? sum[0] : sum[0] + sum[kTiles - 1];
            step.add(s, out);
            __builtin_amdgcn_sched_barrier(0);
            load(t + WAVES, false);
        }

        // join the wavefronts
        l = sum_xor32(sum_xor16(l));
        __syncthreads();
        if (g == 0 && c < HP) room_ml[wave][c] = make_float2(m, l);
#pragma unroll
        for (int i = 0; i < S::kOut; ++i) out[i] *= S::kUnscale;
        S::put(room.sums[wave][c % HP], c, g, out);
        __syncthreads();
        const bool all = t0 == 0 && t1 == units;
        const uint64_t slot = 2ull * blockIdx.x + (t0 == 0 ? 1 : 0);
        constexpr uint32_t kQuads = kDims / 4;
        for (uint32_t i = threadIdx.x; i < heads * kQuads; i += kThreads) {
            const uint32_t r = i / kQuads, quad = i % kQuads;
            if (4 * quad >= a.head_dim) continue;
            float top = neg_inf(), sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) top = fmaxf(top, room_ml[w][r].x);
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float2 ml = room_ml[w][r];
                const float f = ml.x == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);
                sum += f * ml.y;
                o += f * *reinterpret_cast<const f32x4*>(&room.sums[w][r][4 * quad]);
            }
            if (all) {
                f32x4 y;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = sum == 0.0f ? 0.0f : o[j] / sum;
                *reinterpret_cast<f32x4*>(a.output + (line0 + r) * a.head_dim + 4 * quad) = y;
            } else {
                if (quad == 0) a.partial_ml[slot * a.heads + r] = make_float2(top, sum);
                *reinterpret_cast<f32x4*>(a.partial_out + (slot * a.heads + r) * a.head_dim + 4 * quad) = o;
            }
        }
    }
}

hipError_t launch_paged_attention_f32(hipStream_t stream, const PagedAttnParams& a);
hipError_t launch_paged_attention_f16(hipStream_t stream, const PagedAttnParams& a);
hipError_t launch_paged_attention_q8_0(hipStream_t stream, const PagedAttnParams& a);
hipError_t launch_paged_attention_q4_0(hipStream_t stream, const PagedAttnParams& a);

template <int FMT, int NB, int HP>
hipError_t launch_paged_heads(hipStream_t stream, const PagedAttnParams& a) {
    const uint32_t rows = a.sequences * a.kv_heads * a.head_tiles;
    if (a.row_units == 0)
        hipLaunchKernelGGL((paged_attention_kernel<FMT, NB, HP, kPagedAttnWaves, false>), dim3(a.most_parts),
                           dim3(kPagedAttnWaves * kWave), 0, stream, a);
    else if (paged_waves(FMT, NB, a.row_units, rows) == kPagedAttnWaves)
        hipLaunchKernelGGL((paged_attention_kernel<FMT, NB, HP, kPagedAttnWaves, true>), dim3(rows), dim3(kPagedAttnWaves * kWave),
                           0, stream, a);
    else
        hipLaunchKernelGGL((paged_attention_kernel<FMT, NB, HP, paged_row_waves(FMT, NB), true>), dim3(rows),
                           dim3(paged_row_waves(FMT, NB) * kWave), 0, stream, a);
    return hipGetLastError();
}
template <int FMT, int NB>
hipError_t launch_paged_blocks(hipStream_t stream, const PagedAttnParams& a) {
    if constexpr (FMT == kKvQ8_0 || FMT == kKvQ4_0) {
        if (a.group <= 4) return launch_paged_heads<FMT, NB, 4>(stream, a);
        if (a.group <= 8) return launch_paged_heads<FMT, NB, 8>(stream, a);
    }
    return launch_paged_heads<FMT, NB, 16>(stream, a);
}
template <int FMT>
hipError_t launch_paged_format(hipStream_t stream, const PagedAttnParams& a) {
    switch ((a.head_dim + 31) / 32) {
        case 1: return launch_paged_blocks<FMT, 1>(stream, a);
        case 2: return launch_paged_blocks<FMT, 2>(stream, a);
        case 3: return launch_paged_blocks<FMT, 3>(stream, a);
        case 4: return launch_paged_blocks<FMT, 4>(stream, a);
        case 5: return launch_paged_blocks<FMT, 5>(stream, a);
        case 6: return launch_paged_blocks<FMT, 6>(stream, a);
        case 7: return launch_paged_blocks<FMT, 7>(stream, a);
        default: return launch_paged_blocks<FMT, 8>(stream, a);
    }
}

}  // namespace atlas
