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
// p' = 2^{x - m} 2^{ev - m'} with m' about the row's largest x - m + ev, so
// that sum 2^{x - m} v = 2^{m'} sum p' v' keeps every row's precision whatever the
// rows' scales (but a weight below 2^-126, which f32 does not hold, is zero).
// m and m' are whole numbers: all these factors are exact.
//
// A workgroup walks one segment in tiles of KT keys: the tile's rows come from
// the cache as they are stored and are converted once, into the fragments that
// the matrix instructions read (LDS, 16 bytes a lane, in lane order: no bank
// conflicts).  A wavefront holds 16 rows' queries and accumulators in registers
// (32 rows spilled); S^T = K Q^T leaves lane l with query row l % 16, so its
// maximum and sum are the lane's own up to two exchanges, and P^T is the operand
// of O^T = V^T P^T without leaving its registers.
//
// Measured: 64 rows x 100003 keys of 256 dims Q8_0 40 us, of which 12 are start
// and segments; converting and multiplying take about as long as each other.
// 2048 rows x 32768 f32, packed, 192 to 199 us: 1.04 to 1.07 PFLOP/s of f16,
// what a large matrix product reaches here.
#include "prefix_attention.hpp"

namespace atlas {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float max_mag(float a, float b) { return fmaxf(__builtin_fabsf(a), __builtin_fabsf(b)); }

// What a wavefront's lanes have written to LDS is there for its other lanes.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The exponent e that brings a row of largest magnitude `top` to
// [2^14, 2^15) as x 2^-e; rows below 2^-112, whose 2^-e f32 does not hold, only to
// 1 and more, where the pieces have their 22 bits too.
__device__ __forceinline__ int row_exponent(float top) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    return (e < -112 ? -112 : e) - 14;
}

// x times[i] as two f16 vectors, where the product is exact in f32: each piece
// is one instruction, rounded from the exact difference.
struct Pieces {
    half8 hi, lo;
};
template <class Times>
__device__ __forceinline__ Pieces pieces(const float (&x)[8], const Times& times) {
    u32x4_t hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x0 = x[2 * i], x1 = x[2 * i + 1], t0 = times(2 * i), t1 = times(2 * i + 1);
        uint32_t h, l;
        asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(x0), "v"(t0));
        asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(x1), "v"(t1));
        asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(l) : "v"(x0), "v"(t0), "v"(h));
        asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(x1), "v"(t1), "v"(h));
        hi[i] = h;
        lo[i] = l;
    }
    return {__builtin_bit_cast(half8, hi), __builtin_bit_cast(half8, lo)};
}
__device__ __forceinline__ Pieces pieces(const float (&x)[8], float times) {
    return pieces(x, [=](int) { return times; });
}

// A quantised row's exponent is that of its largest block scale and code: the
// pieces keep their bits wherever the row lies in f16's range.
template <int FMT>
constexpr float kMostCode = FMT == kKvQ8_0 ? 128.0f : 8.0f;

// Sizes of a kernel: D the head_dim it is padded to.
template <int D>
struct Wide {
    static constexpr int KT = 32 * 256 / D;  // keys of a tile: 64 KiB of fragments
    static constexpr int KS = D / 32;        // steps of a score
    static constexpr int DT = D / 16;        // blocks of an output row
    static constexpr int KI = KT / 32;       // keys a lane converts
    static constexpr int KU = D / 64;        // units of each
};

template <int D>
struct WideTile {
    half8 key[Wide<D>::KT / 16 * Wide<D>::KS * 2][kWave];    // [16 keys][step][piece]
    half8 value[Wide<D>::KT / 32 * Wide<D>::DT * 2][kWave];  // [32 keys][block][piece]
    int key_exp[Wide<D>::KT];        // of the key row
    int value_exp[Wide<D>::KT];      // of the value row, also as a float
    float value_expf[Wide<D>::KT];
    float value_scale[Wide<D>::KT];  // 2^-value_exp
    float pad[D == 256 ? 128 : 0];       // to whole KiB, for the copies of packed tiles
};

// A lane's part of a tile as loaded: KI * KU key units, 8 keys' value quads.
template <int FMT, int D>
struct RawKeys {
    RawKey<FMT> at[Wide<D>::KI][Wide<D>::KU];
};
template <int FMT>
struct RawValues {
    RawValue<FMT> at[8];
};

// Where this lane's part of a tile lies.
template <int FMT, int D>
struct WideLane {
    uint32_t key_off[Wide<D>::KU][2], value_off;
    uint32_t key_row, value_row;  // first key of each; the others a constant on
    static constexpr uint32_t kQuads = D / 4;
    __device__ WideLane(uint32_t lane, uint32_t wave, uint32_t head_dim) {
#pragma unroll
        for (int u = 0; u < Wide<D>::KU; ++u)
#pragma unroll
            for (uint32_t p = 0; p < 2; ++p) key_off[u][p] = RawKey<FMT>::offset(lane / 8 + 8 * u, head_dim, p);
        key_row = 8 * wave + lane % 8;
        // value groups of 8 keys, kWave / kQuads to a wavefront: of every 32
        // keys, group q has 4 q + {0..3} and 16 more
        const uint32_t group = wave * (kWave / kQuads) + lane / kQuads;
        value_row = 32 * (group / 4) + 4 * (group % 4);
        value_off = RawValue<FMT>::offset(lane % kQuads, head_dim);
    }
};

template <int FMT, int D>
__device__ __forceinline__ void load_keys(RawKeys<FMT, D>& raw, const WideLane<FMT, D>& at, const TileRows<FMT>& t) {
#pragma unroll
    for (int i = 0; i < Wide<D>::KI; ++i)
#pragma unroll
        for (int u = 0; u < Wide<D>::KU; ++u)
            raw.at[i][u].load(t, at.key_row + 32 * i, threadIdx.x % kWave / 8 + 8 * u, at.key_off[u]);
}

template <int FMT, int D>
__device__ __forceinline__ void load_values(RawValues<FMT>& raw, const WideLane<FMT, D>& at, const TileRows<FMT>& t) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        raw.at[j].load(t, at.value_row + 16 * (j >> 2) + (j & 3), threadIdx.x % (D / 4), at.value_off);
}

template <int FMT, int D>
__device__ __forceinline__ void convert_keys(const RawKeys<FMT, D>& raw, WideTile<D>& tile, uint32_t lane, uint32_t wave,
                                             uint32_t left, uint32_t head_dim) {
    using W = Wide<D>;
#pragma unroll
    for (int i = 0; i < W::KI; ++i) {
        float x[W::KU][8], times[W::KU];
        float top = 0.0f;
        const uint32_t key = 32 * i + 8 * wave + lane % 8;
#pragma unroll
        for (int u = 0; u < W::KU; ++u) {
            times[u] = raw.at[i][u].codes(x[u], key < left && 8 * (lane / 8 + 8 * u) < head_dim);
            if (FMT == kKvF32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) top = max_mag(top, x[u][j]);
            } else {
                top = max_mag(top, times[u] * kMostCode<FMT>);
            }
        }
        top = max_xor32(max_xor16(max_xor8(top)));
        const int e = row_exponent(top);
        const float scale = pow2i(-e);
        if (lane < 8) tile.key_exp[key] = e;
#pragma unroll
        for (int u = 0; u < W::KU; ++u) {
            const Pieces p = pieces(x[u], times[u] * scale);
            const uint32_t unit = lane / 8 + 8 * u;
            const uint32_t frag = (key / 16 * W::KS + unit / 4) * 2, to = unit % 4 * 16 + key % 16;
            tile.key[frag][to] = p.hi;
            tile.key[frag + 1][to] = p.lo;
        }
    }
}

template <int FMT, int D>
__device__ __forceinline__ void convert_values(const RawValues<FMT>& raw, WideTile<D>& tile, uint32_t lane, uint32_t wave,
                                               uint32_t left, uint32_t head_dim) {
    using W = Wide<D>;
    constexpr uint32_t kQuads = D / 4;
    const uint32_t group = wave * (kWave / kQuads) + lane / kQuads, quad = lane % kQuads;
    const uint32_t key0 = 32 * (group / 4) + 4 * (group % 4);
    float x[8][4], times[8];  // [key][dim]
    float top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        times[j] = raw.at[j].codes(x[j], key0 + 16 * (j >> 2) + (j & 3) < left && 4 * quad < head_dim);
        top[j] = FMT == kKvF32 ? fmaxf(max_mag(x[j][0], x[j][1]), max_mag(x[j][2], x[j][3])) : __builtin_fabsf(times[j] * kMostCode<FMT>);
    }
    // eight maxima over the group's lanes: each step halves what a lane keeps,
    // ending with key lane % 8
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
        const uint32_t key = key0 + 16 * (quad / 4) + quad % 4;
        const int e = row_exponent(m);
        // a row of zeros raises no m', or it could leave the other rows no bits
        const bool zeros = m == 0.0f;
        tile.value_exp[key] = zeros ? -1000 : e;
        tile.value_expf[key] = zeros ? neg_inf() : static_cast<float>(e);
        // an infinity would leave the row's other values no bits: NaN, not a wrong number
        tile.value_scale[key] = m == __builtin_inff() ? __builtin_nanf("") : pow2i(-e);
    }
    wave_lds_fence();
    const f32x4 s0 = *reinterpret_cast<const f32x4*>(&tile.value_scale[key0]);
    const f32x4 s1 = *reinterpret_cast<const f32x4*>(&tile.value_scale[key0 + 16]);
#pragma unroll
    for (int j = 0; j < 8; ++j) times[j] *= j < 4 ? s0[j & 3] : s1[j & 3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float y[8] = {x[0][e], x[1][e], x[2][e], x[3][e], x[4][e], x[5][e], x[6][e], x[7][e]};
        const Pieces p = pieces(y, [&](int j) { return times[j]; });
        // dim e of quad q: row q % 16 of block 4 (q / 16) + e
        const uint32_t frag = (group / 4 * W::DT + 4 * (quad / 16) + e) * 2, to = group % 4 * 16 + quad % 16;
        tile.value[frag][to] = p.hi;
        tile.value[frag + 1][to] = p.lo;
    }
}

__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The products read their fragments two steps of four ahead: left to itself
// the compiler saves the registers and waits for every read (LDS latency, not
// its rate, then set the time: 32768 x 2048 rows 343 us).
template <int D>
__device__ __forceinline__ void score_pair(const WideTile<D>& tile, int t, uint32_t lane, const half8 (&q_hi)[Wide<D>::KS],
                                           const half8 (&q_lo)[Wide<D>::KS], int q_exp, f32x4& s0, f32x4& s1) {
    constexpr int kSteps = Wide<D>::KS;
    half8 f[2][4];
    auto read = [&](int k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[k % 2][i] = tile.key[((t + i / 2) * kSteps + k) * 2 + i % 2][lane];
    };
    s0 = s1 = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    __builtin_amdgcn_sched_barrier(0);
    read(0);
    read(1);
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        half8(&g)[4] = f[k % 2];
        s0 = mfma(g[1], q_hi[k], s0);
        s1 = mfma(g[3], q_hi[k], s1);
        s0 = mfma(g[0], q_lo[k], s0);
        s1 = mfma(g[2], q_lo[k], s1);
        s0 = mfma(g[0], q_hi[k], s0);
        s1 = mfma(g[2], q_hi[k], s1);
        __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
        if (k + 2 < kSteps) {
            read(k + 2);
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    // the key rows' exponents belong to the keys: read before the barrier
    // behind which the next tile's may be written
    const i32x4 e0 = *reinterpret_cast<const i32x4*>(&tile.key_exp[16 * t + lane / 16 * 4]);
    const i32x4 e1 = *reinterpret_cast<const i32x4*>(&tile.key_exp[16 * t + 16 + lane / 16 * 4]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        s0[j] = __builtin_ldexpf(s0[j], e0[j] + q_exp);
        s1[j] = __builtin_ldexpf(s1[j], e1[j] + q_exp);
    }
}

template <int D>
__device__ __forceinline__ void add_values(const WideTile<D>& tile, int b, uint32_t lane, const Pieces& p,
                                           f32x4 (&out)[Wide<D>::DT]) {
    constexpr int kSteps = Wide<D>::DT / 2;
    half8 f[2][4];
    auto read = [&](int k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[k % 2][i] = tile.value[(b * 2 * kSteps + 2 * k + i / 2) * 2 + i % 2][lane];
    };
    __builtin_amdgcn_sched_barrier(0);
    read(0);
    read(1);
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        half8(&g)[4] = f[k % 2];
        f32x4 &o0 = out[2 * k], &o1 = out[2 * k + 1];
        o0 = mfma(g[1], p.hi, o0);
        o1 = mfma(g[3], p.hi, o1);
        o0 = mfma(g[0], p.lo, o0);
        o1 = mfma(g[2], p.lo, o1);
        o0 = mfma(g[0], p.hi, o0);
        o1 = mfma(g[2], p.hi, o1);
        __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
        if (k + 2 < kSteps) {
            read(k + 2);
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
}

// Which rows and which part of the prompt a workgroup takes.  Workgroups go to
// the eight XCDs in turn; each XCD gets a run of items, whose segments its L2 then
// reads once or shares with one neighbour (whole segments to an XCD, plain
// order, and so: 800 rows x 8192 f32 56, 66 and 56 us, 1440 rows 78, 75 and 71,
// 1092 rows x 5979 51, 40 and 41).
struct WideItem {
    uint32_t slot, tile, kv_head, begin, end;
    bool none;
    static __host__ __device__ uint32_t grid(uint32_t items) { return (items + 7) / 8 * 8; }
    __device__ WideItem(const AttnParams& a, uint32_t kt) {
        const uint32_t items = a.prefix_tiles * a.prefix_slots * a.kv_heads;
        uint32_t item = blockIdx.x % 8 * (grid(items) / 8) + blockIdx.x / 8;
        none = item >= items;
        tile = item % a.prefix_tiles;
        item /= a.prefix_tiles;
        slot = item % a.prefix_slots;
        kv_head = item / a.prefix_slots;
        // the divisions leave them in vector registers; buffers' bases hang on them
        slot = __builtin_amdgcn_readfirstlane(slot);
        tile = __builtin_amdgcn_readfirstlane(tile);
        kv_head = __builtin_amdgcn_readfirstlane(kv_head);
        part_of(a.prefix_length, kt, slot, a.prefix_slots, begin, end);
    }
};

// 16 query rows of a wavefront as operands, lane (row n, quarter) holding the
// dims of units 4 s + quarter, and what they have summed.
template <int FMT, int D, bool RUNS>
struct WideRows {
    half8 q_hi[Wide<D>::KS], q_lo[Wide<D>::KS];
    int q_exp;
    f32x4 out[Wide<D>::DT];
    // Whole numbers; every x <= m + 8 and x - m + ev <= mv + 8, so a weight
    // 2^(x - m) is at most 2^8 and p' = 2^(x - m + ev - mv + 6) at most 2^14.  mv is
    // counted from m: a score may be so large that its neighbours lie further
    // apart than the exponents of values.
    float m, mv, l;
    // below it a result is zero, whatever the values
    static constexpr float kLeast = -200.0f;
    // sums of the runs that have ended, if any, relative to the m and mv of then
    bool ended;
    f32x4 out_before[Wide<D>::DT];
    float m_before, mv_before, l_before;

    __device__ __forceinline__ WideRows(const AttnParams& a, uint32_t kv_head, uint32_t row, uint32_t quarter) {
        const uint32_t at = min(row, a.rows - 1);
        const float* q_row =
            a.q + (static_cast<uint64_t>(at / a.group) * a.q_heads + kv_head * a.group + at % a.group) * a.head_dim;
        float x[Wide<D>::KS][8];
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < Wide<D>::KS; ++s) {
            load_query8<FMT>(q_row, 4 * s + quarter, a.head_dim, a.scale, x[s]);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max_mag(top, x[s][j]);
        }
        top = max_xor32(max_xor16(top));
        q_exp = row_exponent(top);
        const float scale = pow2i(-q_exp);
#pragma unroll
        for (int s = 0; s < Wide<D>::KS; ++s) {
            const Pieces p = pieces(x[s], scale);
            q_hi[s] = p.hi;
            q_lo[s] = p.lo;
        }
#pragma unroll
        for (int d = 0; d < Wide<D>::DT; ++d) out[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m = -0x1.fffffep127f;  // the least number, so that differences of m are never NaN
        mv = kLeast;
        l = 0.0f;
        ended = false;
    }

    // The sums so far put aside.  Adding key after key to one f32 rounds every
    // time, and with keys alike every time the same way: the results of 60001 equal
    // keys came to 4e-4 too much.  From every 32 keys a lane's l takes one sum of eight
    // weights and an accumulator three products; so a run of 512 keys rounds 16 and
    // 48 times, a segment of kMostPromptKeys its runs 128 times: off by 5.2e-6 for
    // equal keys.  A segment of at most kShort keys is one run (off by 6.8e-6) of a
    // kernel without RUNS, whose registers and code they lengthen (100003 keys, 64
    // rows: 51.3 us, without 50.5).
    static constexpr uint32_t kRun = 512, kShort = 1024;
    __device__ __forceinline__ void end_run() {
        join_runs();
        l_before = l;
        l = 0.0f;
        m_before = m;
        mv_before = mv;
#pragma unroll
        for (int d = 0; d < Wide<D>::DT; ++d) {
            out_before[d] = out[d];
            out[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        ended = true;
    }
    __device__ __forceinline__ void join_runs() {
        if (!RUNS || __builtin_expect(!ended, 1)) return;
        const float down = m_before - m;
        const float fade = __builtin_amdgcn_exp2f(down), fade_v = __builtin_amdgcn_exp2f(down + (mv_before - mv));
        l += l_before * fade;
#pragma unroll
        for (int d = 0; d < Wide<D>::DT; ++d) out[d] += out_before[d] * fade_v;
    }

    // Block b of 32 keys: scores to weights, and their values added.  Register
    // j of a score: key 32 b + 16 (j / 4) + 4 quarter + j % 4 of the tile, of
    // which `left` are there.
    __device__ __forceinline__ void add(const WideTile<D>& tile, int b, const f32x4& s0, const f32x4& s1, uint32_t left,
                                        uint32_t lane) {
        const uint32_t quarter = lane / 16;
        float s[8];
        f32x4 evf[2];
        i32x4 ev[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t key = 32 * b + 16 * t + 4 * quarter;
            evf[t] = *reinterpret_cast<const f32x4*>(&tile.value_expf[key]);
            ev[t] = *reinterpret_cast<const i32x4*>(&tile.value_exp[key]);
        }
        const auto score = [&](int j) {
            const float x = j < 4 ? s0[j] : s1[j - 4];
            return left < Wide<D>::KT && 32 * b + 16 * (j / 4) + 4 * quarter + j % 4 >= left ? neg_inf() : x;
        };
        float top = neg_inf(), top_v = neg_inf();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j] = score(j) - m;
            top = fmaxf(top, s[j]);
            top_v = fmaxf(top_v, s[j] + evf[j / 4][j % 4]);
        }
        top = max_xor32(max_xor16(top));
        top_v = max_xor32(max_xor16(top_v));
        if (__builtin_amdgcn_ballot_w64(top > 8.0f || top_v > mv + 8.0f) != 0) raise(score, evf, s);
        const int shift = 6 - static_cast<int>(mv);
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = __builtin_amdgcn_exp2f(s[j]);
            s[j] = __builtin_ldexpf(w[j], ev[j / 4][j % 4] + shift);
        }
        l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        add_values<D>(tile, b, lane, pieces(s, 1.0f), out);
    }

    // New m and mv, and the differences from the scores again.
    template <class Score>
    __device__ __forceinline__ void raise(const Score& score, const f32x4 (&evf)[2], float (&s)[8]) {
        float top = neg_inf(), top_v = neg_inf();
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, score(j));
        const float m_new = fmaxf(m, __builtin_ceilf(max_xor32(max_xor16(top)))), down = m - m_new;
        m = m_new;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j] = score(j) - m;
            top_v = fmaxf(top_v, s[j] + evf[j / 4][j % 4]);
        }
        const float mv_new = fmaxf(fmaxf(mv + down, __builtin_ceilf(max_xor32(max_xor16(top_v)))), kLeast);
        const float fade = __builtin_amdgcn_exp2f(mv + down - mv_new);
        l *= __builtin_amdgcn_exp2f(down);
        mv = mv_new;
#pragma unroll
        for (int d = 0; d < Wide<D>::DT; ++d) out[d] *= fade;
    }

    // The segment's sums, relative to 2^m, by way of LDS (`room` of the
    // wavefront, 8 rows at a time) so that whole rows are written: straight from
    // the accumulators, 16 bytes here and there, it took 13 us.
    static constexpr uint32_t kPitch = D + 4, kRoom = 8 * kPitch;
    __device__ __forceinline__ void finish(const AttnParams& a, const WideItem& item, uint32_t row0, float* room, uint32_t lane) {
        const uint32_t n = lane % 16, quarter = lane / 16;
        join_runs();
        const float all = sum_xor32(sum_xor16(l));
        const int back = static_cast<int>(mv) - 6;
        const uint64_t to = (static_cast<uint64_t>(item.slot) * a.kv_heads + item.kv_head) * a.rows + row0;
        if (quarter == 0 && row0 + n < a.rows) a.partial_ml[to + n] = make_float2(m, all);
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
            if (n / 8 == half) {
#pragma unroll
                for (int d = 0; d < Wide<D>::DT; d += 4)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f32x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = __builtin_ldexpf(out[d + e][i], back);
                        put_quad<FMT>(room + n % 8 * kPitch, 4 * d + 4 * quarter + i, v);
                    }
            }
            wave_lds_fence();
            constexpr uint32_t kQuads = D / 4, kAtOnce = kWave / kQuads;
            const uint32_t quad = lane % kQuads;
#pragma unroll
            for (uint32_t r0 = 0; r0 < 8; r0 += kAtOnce) {
                const uint32_t r = r0 + lane / kQuads, row = 8 * half + r;
                const f32x4 v = *reinterpret_cast<const f32x4*>(room + r * kPitch + 4 * quad);
                if (row0 + row < a.rows && 4 * quad < a.head_dim)
                    *reinterpret_cast<f32x4*>(a.partial_out + (to + row) * a.head_dim + 4 * quad) = v;
            }
            wave_lds_fence();
        }
    }
};

// Eight wavefronts: four convert a tile while the other four, 16 rows each,
// multiply the one before it, so that the vector units and the matrix units of
// every SIMD have a wavefront of their own (all eight doing both in turn, in two
// workgroups, 48 us for 100003 keys and 64 rows; so 43).  One barrier a tile:
// behind it the converted tile is there and the buffer of the one before is
// free.
constexpr int kWideThreads = 512;

template <int FMT, int D, bool RUNS>
__global__ __launch_bounds__(kWideThreads, 2) void attn_wide_kernel(AttnParams a) {
    using W = Wide<D>;
    __shared__ WideTile<D> buffers[2];
    const uint32_t lane = threadIdx.x % kWave, n = lane % 16, quarter = lane / 16;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    const WideItem item(a, W::KT);
    if (item.none) return;
    const uint32_t end = item.end;
    uint32_t buffer = 0;
    if (wave >= 4) {
        __builtin_amdgcn_s_setprio(2);  // converting takes longest: 43.2 us without (100003 keys, 64 rows)
        const uint32_t head_off = static_cast<uint32_t>(head_offset<FMT>(item.kv_head, a.head_dim));
        const uint8_t* keys = a.prefix + head_off;
        const uint8_t* values = a.prefix + a.prefix_plane + head_off;
        const WideLane<FMT, D> mine(lane, wave - 4, a.head_dim);
        const auto rows_of = [&](const uint8_t* plane, uint32_t first) {
            const uint32_t there = first < end ? min(end - first, static_cast<uint32_t>(W::KT)) : 0u;
            return TileRows<FMT>(plane, there ? first : end - 1, there, a.row_bytes, head_off);
        };
        // a tile of f32 rows is enough in flight, of quantised ones two are
        constexpr int kAhead = FMT == kKvF32 ? 1 : 2;
        RawKeys<FMT, D> raw_keys[kAhead];
        RawValues<FMT> raw_values[kAhead];
        uint32_t first = item.begin;
        if (first < end) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                load_keys(raw_keys[i], mine, rows_of(keys, first + i * W::KT));
                load_values(raw_values[i], mine, rows_of(values, first + i * W::KT));
            }
        }
        while (first < end) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (first >= end) break;
                convert_keys(raw_keys[i], buffers[buffer], lane, wave - 4, end - first, a.head_dim);
                load_keys(raw_keys[i], mine, rows_of(keys, first + kAhead * W::KT));
                convert_values(raw_values[i], buffers[buffer], lane, wave - 4, end - first, a.head_dim);
                load_values(raw_values[i], mine, rows_of(values, first + kAhead * W::KT));
                __syncthreads();
                first += W::KT;
                buffer ^= 1;
            }
        }
        return;
    }
    const uint32_t row0 = item.tile * 64 + wave * 16;
    const bool busy = row0 < a.rows;  // the wavefront has rows
    WideRows<FMT, D, RUNS> rows(a, item.kv_head, row0 + n, quarter);
    for (uint32_t first = item.begin; first < end; first += W::KT, buffer ^= 1) {
        __syncthreads();
        if (!busy) continue;
        if (RUNS && __builtin_expect(first != item.begin && (first - item.begin) % rows.kRun == 0, 0)) rows.end_run();
        const WideTile<D>& tile = buffers[buffer];
        f32x4 scores[W::KT / 16];
#pragma unroll
        for (int t = 0; t < W::KT / 16; t += 2)
            score_pair<D>(tile, t, lane, rows.q_hi, rows.q_lo, rows.q_exp, scores[t], scores[t + 1]);
#pragma unroll
        for (int b = 0; b < W::KT / 32; ++b) rows.add(tile, b, scores[2 * b], scores[2 * b + 1], end - first, lane);
    }
    // the buffer of the tile before the last is free
    if (busy) rows.finish(a, item, row0, reinterpret_cast<float*>(&buffers[buffer]) + wave * rows.kRoom, lane);
}

// The prompt's tiles converted once, for batches whose rows would have every
// one converted many times: a workgroup a tile of a KV head.  Its bytes bound
// it: 32768 keys of 256 dims f32 26 us, 5.2 TB/s read and written.
template <int FMT, int D>
__global__ __launch_bounds__(kAttnThreads) void attn_pack_kernel(AttnParams a, WideTile<D>* packed, uint32_t tiles) {
    using W = Wide<D>;
    __shared__ WideTile<D> tile;
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    const uint32_t kv_head = __builtin_amdgcn_readfirstlane(blockIdx.x / tiles);
    const uint32_t first = __builtin_amdgcn_readfirstlane(blockIdx.x % tiles) * W::KT;
    const uint32_t head_off = static_cast<uint32_t>(head_offset<FMT>(kv_head, a.head_dim));
    const WideLane<FMT, D> mine(lane, wave, a.head_dim);
    RawKeys<FMT, D> raw_keys;
    RawValues<FMT> raw_values;
    const uint32_t there = min(a.prefix_length - first, static_cast<uint32_t>(W::KT));
    load_keys(raw_keys, mine, TileRows<FMT>(a.prefix + head_off, first, there, a.row_bytes, head_off));
    load_values(raw_values, mine, TileRows<FMT>(a.prefix + a.prefix_plane + head_off, first, there, a.row_bytes, head_off));
    convert_keys(raw_keys, tile, lane, wave, there, a.head_dim);
    convert_values(raw_values, tile, lane, wave, there, a.head_dim);
    __syncthreads();
    const f32x4* from = reinterpret_cast<const f32x4*>(&tile);
    f32x4* to = reinterpret_cast<f32x4*>(packed + blockIdx.x);
    for (uint32_t i = threadIdx.x; i < sizeof(tile) / 16; i += kAttnThreads) to[i] = from[i];
}

// Packed tiles: eight wavefronts of 16 rows, tiles copied to LDS one ahead
// (no registers, no conversion), one barrier a tile.
constexpr int kPackedThreads = 512;

template <int FMT, int D>
__global__ __launch_bounds__(kPackedThreads, 2) void attn_packed_kernel(AttnParams a, const WideTile<D>* packed, uint32_t tiles) {
    using W = Wide<D>;
    static_assert(sizeof(WideTile<D>) >= 8 * WideRows<FMT, D, true>::kRoom * sizeof(float), "eight wavefronts' rows fit a buffer");
    static_assert(sizeof(WideTile<D>) % 1024 == 0, "copied by whole KiB");
    constexpr uint32_t kChunks = sizeof(WideTile<D>) / 1024;
    __shared__ WideTile<D> buffers[2];
    const uint32_t lane = threadIdx.x % kWave, n = lane % 16, quarter = lane / 16;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    const WideItem item(a, W::KT);
    if (item.none) return;
    const uint32_t row0 = item.tile * 128 + wave * 16, row = row0 + n, end = item.end;
    const bool busy = row0 < a.rows;
    const WideTile<D>* source = packed + static_cast<uint64_t>(item.kv_head) * tiles;
    const uint32_t lds = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)(&buffers[0])));
    auto copy = [&](uint32_t first, uint32_t buffer) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(source + first / W::KT);
#pragma unroll
        for (uint32_t c = 0; c < (kChunks + 7) / 8; ++c) {
            const uint32_t chunk = c * 8 + wave;
            // 64 lanes of 16 bytes to LDS at M0, an output of the asm so that the
            // compiler knows of its change; nothing comes back to a register
            uint32_t m0;
            if (chunk < kChunks)
                asm volatile("s_mov_b32 %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3"
                             : "={m0}"(m0)
                             : "s"(lds + buffer * static_cast<uint32_t>(sizeof(WideTile<D>)) + chunk * 1024),
                               "v"(lane * 16), "s"(from + chunk * 1024)
                             : "memory");
        }
    };
    if (item.begin < end) copy(item.begin, 0);
    WideRows<FMT, D, true> rows(a, item.kv_head, row, quarter);
    uint32_t buffer = 0;
    for (uint32_t first = item.begin; first < end; first += W::KT, buffer ^= 1) {
        // this tile has arrived, and every wavefront is done with the one before
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (first + W::KT < end) copy(first + W::KT, buffer ^ 1);
        if (!busy) continue;
        if (__builtin_expect(first != item.begin && (first - item.begin) % rows.kRun == 0, 0)) rows.end_run();
        const uint32_t left = end - first;
        const WideTile<D>& tile = buffers[buffer];
        f32x4 scores[W::KT / 16];
#pragma unroll
        for (int t = 0; t < W::KT / 16; t += 2)
            score_pair<D>(tile, t, lane, rows.q_hi, rows.q_lo, rows.q_exp, scores[t], scores[t + 1]);
#pragma unroll
        for (int b = 0; b < W::KT / 32; ++b) rows.add(tile, b, scores[2 * b], scores[2 * b + 1], left, lane);
    }
    // the buffer of the tile before the last is free
    if (busy) rows.finish(a, item, row0, reinterpret_cast<float*>(&buffers[buffer]) + wave * rows.kRoom, lane);
}

template <int FMT, int D>
hipError_t launch_wide(hipStream_t stream, uint32_t items, const AttnParams& a, void* room) {
    if (!room) {
        const uint32_t tiles = (a.prefix_length + Wide<D>::KT - 1) / Wide<D>::KT;
        const uint32_t longest = (tiles + a.prefix_slots - 1) / a.prefix_slots * Wide<D>::KT;
        const dim3 grid(WideItem::grid(items)), block(kWideThreads);
        if (longest <= WideRows<FMT, D, false>::kShort)
            hipLaunchKernelGGL((attn_wide_kernel<FMT, D, false>), grid, block, 0, stream, a);
        else
            hipLaunchKernelGGL((attn_wide_kernel<FMT, D, true>), grid, block, 0, stream, a);
        return hipGetLastError();
    }
    WideTile<D>* packed = static_cast<WideTile<D>*>(room);
    const uint32_t tiles = (a.prefix_length + Wide<D>::KT - 1) / Wide<D>::KT;
    hipLaunchKernelGGL((attn_pack_kernel<FMT, D>), dim3(tiles * a.kv_heads), dim3(kAttnThreads), 0, stream, a, packed, tiles);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // packed tiles of f32 and Q8_0 rows have one order of dims
    constexpr int kOrder = FMT == kKvQ4_0 ? kKvQ4_0 : kKvF32;
    hipLaunchKernelGGL((attn_packed_kernel<kOrder, D>), dim3(WideItem::grid(items)), dim3(kPackedThreads), 0, stream, a, packed, tiles);
    return hipGetLastError();
}

template <int FMT>
hipError_t launch_wide(hipStream_t stream, uint32_t items, const AttnParams& a, void* room) {
    if (a.head_dim <= 64) return launch_wide<FMT, 64>(stream, items, a, room);
    if (a.head_dim <= 128) return launch_wide<FMT, 128>(stream, items, a, room);
    return launch_wide<FMT, 256>(stream, items, a, room);
}

}  // namespace

uint64_t attn_packed_bytes(uint32_t head_dim, uint32_t kv_heads, uint32_t prefix_length) {
    const uint32_t d = head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256), kt = 32 * 256 / d;
    const uint64_t tile = d == 64 ? sizeof(WideTile<64>) : (d == 128 ? sizeof(WideTile<128>) : sizeof(WideTile<256>));
    return (static_cast<uint64_t>(prefix_length) + kt - 1) / kt * kv_heads * tile;
}

hipError_t launch_attn_wide(hipStream_t stream, int format, uint32_t items, const AttnParams& a, void* room) {
    if (format == kKvF32) return launch_wide<kKvF32>(stream, items, a, room);
    if (format == kKvQ8_0) return launch_wide<kKvQ8_0>(stream, items, a, room);
    return launch_wide<kKvQ4_0>(stream, items, a, room);
}

}  // namespace atlas
