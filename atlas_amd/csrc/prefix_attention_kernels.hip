// prefix_attention_kernels.hip -- attention of a batch's new tokens over a
// prompt that all sequences share and over each sequence's own cache, reading
// the caches that the KV append writes ([K | V][position][row]; f32, Q8_0 or
// Q4_0 rows).  No counterpart in the reference, whose executors decode one
// sequence.
//
// For query head h of token t of sequence b, with KV head h / group:
//   x_j = scale * (q . k_j) over the prompt's rows and own rows
//         j < len_b - (tokens - 1 - t),
//   out = sum_j e^{x_j} v_j / sum_j e^{x_j}, zero where nothing is seen.
// The sum over j is split into segments (parts of the prompt, parts of the
// sequence's own rows); a segment leaves its maximum m, its sum l of 2^{x - m}
// and its sum O of 2^{x - m} v, and a second launch joins a row's segments:
// out = sum_s 2^{m_s - M} O_s / sum_s 2^{m_s - M} l_s.  The prompt's segments
// hold the rows of all sequences, so its cache is read once for the batch.
#include "prefix_attention.hpp"

namespace atlas {
namespace {

// The blocks of dims whose products with 16 keys are summed at once.
constexpr int kAtOnce = 4;

// sum += the products of the keys that a row sees, key by key, from block `block` on: for
// the tiles where a key that only some rows see holds values that are no numbers.
template <int NG>
__device__ __forceinline__ void add_seen(const float (&v)[4][NG * 4], const float (&p)[4], int block, uint32_t key0,
                                         uint32_t seen, f32x4 (&sum)[kAtOnce]) {
    const uint32_t lane = threadIdx.x % kWave, n = lane % 16, quarter = lane / 16;
    for (uint32_t from = 0; from < 4; ++from)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool sees = key0 + 4 * from + r < seen;
            const float weight = __shfl(p[r], static_cast<int>(n + 16 * from), kWave);
#pragma unroll
            for (int g = 0; g < kAtOnce; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = __shfl(v[r][block + g], static_cast<int>(4 * quarter + i + 16 * from), kWave);
                    sum[g][i] = sees ? sum[g][i] + weight * x : sum[g][i];
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
}

// What a lane of the own rows' kernel holds of a key: NB units of 8 dims,
// `quarter` of four lanes; and of a value: NG quads, lane n of 16.  Any order of
// the dims will do that queries and outputs share.  Of f32 rows a load is 16 bytes
// and neighbouring lanes have neighbouring units; of quantised rows a lane's
// units are neighbours, so that a few wide loads bring them (by loads of 2 and 4
// bytes 24 sequences with 5 drafts, Q4_0, took 27 us, so 23).
template <int FMT, int NB>
struct KeyRun {
    static constexpr int kUnit = FMT == kKvQ8_0 ? 8 : 4, kBlock = FMT == kKvQ8_0 ? 34 : 18;  // bytes
    static constexpr int kBlocks = NB < 4 ? 1 : NB / 4, kWords = NB * kUnit / 4 / kBlocks;    // words of each block
    uint32_t c[kBlocks][kWords];
    uint16_t d[kBlocks];
    static __device__ uint32_t unit(uint32_t quarter, uint32_t b) { return NB * quarter + b; }
    __device__ __forceinline__ void load(const TileRows<FMT>& t, uint32_t row, uint32_t quarter, uint32_t head_dim) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            const uint32_t block = unit(quarter, 0) / 4 + i, off = 32 * block < head_dim ? block * kBlock : 0u;
            const uint32_t behind = 2 + (NB < 4 ? unit(quarter, 0) % 4 * kUnit : 0);
            d[i] = t.template at<uint16_t>(row, off, 0);
            if constexpr (kWords == 2) {
                const u32x2_a2 w = t.template at<u32x2_a2>(row, off, behind);
                c[i][0] = w.x;
                c[i][1] = w.y;
            } else {
#pragma unroll
                for (int k = 0; k < kWords; k += 4) {
                    const u32x4_a2 w = t.template at<u32x4_a2>(row, off, behind + 4 * k);
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[i][k + j] = w[j];
                }
            }
        }
    }
    __device__ __forceinline__ void values(int b, uint32_t quarter, uint32_t head_dim, bool there, float (&v)[8]) const {
        const int i = b / 4, w = b % 4 * (kUnit / 4);
        RawKey<FMT> raw;
        if constexpr (FMT == kKvQ8_0)
            raw.c = u32x2_t{c[i][w], c[i][w + 1]};
        else
            raw.c = c[i][w];
        raw.d = d[i];
        raw_values(raw, v, there && 8 * unit(quarter, b) < head_dim);
    }
};
template <int NB>
struct KeyRun<kKvF32, NB> {
    RawKey<kKvF32> k[NB];
    static __device__ uint32_t unit(uint32_t quarter, uint32_t b) { return 4 * b + quarter; }
    __device__ __forceinline__ void load(const TileRows<kKvF32>& t, uint32_t row, uint32_t quarter, uint32_t head_dim) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint32_t u = unit(quarter, b);
            const uint32_t off[2] = {RawKey<kKvF32>::offset(u, head_dim, 0), RawKey<kKvF32>::offset(u, head_dim, 1)};
            k[b].load(t, row, u, off);
        }
    }
    __device__ __forceinline__ void values(int b, uint32_t, uint32_t, bool, float (&v)[8]) const { raw_values(k[b], v, true); }
};
template <int FMT, int NG>
struct ValueRun {
    static constexpr uint32_t kQuad = FMT == kKvQ8_0 ? 4 : 2, kBlock = FMT == kKvQ8_0 ? 34 : 18;  // bytes
    static constexpr int kWords = NG * kQuad < 4 ? 1 : NG * kQuad / 4;
    uint32_t c[kWords];
    uint16_t d;
    static __device__ uint32_t quad(uint32_t n, uint32_t g) { return NG * n + g; }
    __device__ __forceinline__ void load(const TileRows<FMT>& t, uint32_t row, uint32_t n, uint32_t head_dim) {
        const uint32_t q = quad(n, 0), off = 4 * q < head_dim ? q / 8 * kBlock : 0u, behind = 2 + q % 8 * kQuad;
        d = t.template at<uint16_t>(row, off, 0);
        if constexpr (NG * kQuad == 2) {
            c[0] = t.template at<uint16_t>(row, off, behind);
        } else if constexpr (kWords == 1) {
            c[0] = t.template at<u32_a2>(row, off, behind);
        } else if constexpr (kWords == 2) {
            const u32x2_a2 w = t.template at<u32x2_a2>(row, off, behind);
            c[0] = w.x;
            c[1] = w.y;
        } else {
            const u32x4_a2 w = t.template at<u32x4_a2>(row, off, behind);
#pragma unroll
            for (int j = 0; j < 4; ++j) c[j] = w[j];
        }
    }
    __device__ __forceinline__ void values(int g, uint32_t n, uint32_t head_dim, bool there, float (&v)[4]) const {
        RawValue<FMT> raw;
        if constexpr (FMT == kKvQ8_0)
            raw.c = c[g];
        else
            raw.c = static_cast<uint16_t>(c[g / 2] >> (16 * (g % 2)));
        raw.d = d;
        raw_values(raw, v, there && 4 * quad(n, g) < head_dim);
    }
};
template <int NG>
struct ValueRun<kKvF32, NG> {
    RawValue<kKvF32> v4[NG];
    static __device__ uint32_t quad(uint32_t n, uint32_t g) { return 16 * g + n; }
    __device__ __forceinline__ void load(const TileRows<kKvF32>& t, uint32_t row, uint32_t n, uint32_t head_dim) {
#pragma unroll
        for (int g = 0; g < NG; ++g) v4[g].load(t, row, quad(n, g), RawValue<kKvF32>::offset(quad(n, g), head_dim));
    }
    __device__ __forceinline__ void values(int g, uint32_t, uint32_t, bool, float (&v)[4]) const { raw_values(v4[g], v, true); }
};

// One workgroup: 16 query rows of one KV head against one segment of a
// sequence's own rows (or of the prompt, for batches of up to 16 rows).  Its
// bytes bound it over long caches (64 sequences of up to 8192 rows of 256 dims,
// 0.6 GB: 147 us, 4.1 TB/s), start and join over short ones.  More rows go by
// more workgroups: two tiles of 16 in one took 38 us where two workgroups take
// 23 (64 sequences, 4 tokens of 8 heads, 256 dims).  The wavefronts take its
// keys 16 at a time in turn, straight from the cache into the operands'
// registers, with the next 16 loading while these are used.  Products are
// v_mfma_f32_16x16x4 (f32 throughout): S^T = K Q^T leaves lane l with query row
// l % 16 and keys 4 (l / 16) + r, which is the operand that O^T = V^T P^T wants,
// so P never leaves its registers and a row's statistics are the lane's own.
// Queries wait in LDS.
template <int FMT, int NB>
__global__ __launch_bounds__(kAttnThreads, NB < 8 ? 3 : (FMT == kKvF32 ? 1 : 2)) void attn_rows_kernel(AttnParams a) {
    constexpr int NG = (NB + 1) / 2;  // groups of 64 dims
    constexpr uint32_t kDims = 64 * NG, kPitch = kDims + 4;
    static_assert(kAttnWaves * 16 * kPitch * sizeof(float) >= NB * 2 * kWave * sizeof(f32x4), "the queries fit");
    // queries [step][half][lane]; at the end the wavefronts' sums, row by row
    __shared__ union {
        f32x4 queries[NB * 2][kWave];
        float sums[kAttnWaves][16][kPitch];
    } room;
    __shared__ float2 room_ml[kAttnWaves][16];
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    const uint32_t n = lane % 16, quarter = lane / 16;

    // which rows, which keys
    uint32_t item = blockIdx.x;
    const bool shared = item < a.prefix_items;
    uint32_t kv_head, row0, row_end, slot, key_begin, key_end, length = 0, seq = 0;
    const uint8_t *keys, *values;
    if (shared) {
        const uint32_t tile = item % a.prefix_tiles;
        item /= a.prefix_tiles;
        slot = item % a.prefix_slots;
        kv_head = __builtin_amdgcn_readfirstlane(item / a.prefix_slots);
        row0 = tile * 16;
        row_end = a.rows;
        part_of(a.prefix_length, 64, slot, a.prefix_slots, key_begin, key_end);
        keys = a.prefix;
        values = a.prefix + a.prefix_plane;
    } else {
        item -= a.prefix_items;
        const uint32_t tile = item % a.own_tiles;
        item /= a.own_tiles;
        const uint32_t part_index = item % a.own_slots;
        item /= a.own_slots;
        kv_head = __builtin_amdgcn_readfirstlane(item % a.kv_heads);
        seq = __builtin_amdgcn_readfirstlane(item / a.kv_heads);
        slot = a.prefix_slots + part_index;
        row0 = seq * a.seq_rows + tile * 16;
        row_end = (seq + 1) * a.seq_rows;
        length = min(a.lengths[seq], a.capacity);
        part_of(length, 64, part_index, a.own_slots, key_begin, key_end);
        const uint64_t base = static_cast<uint64_t>(seq) * a.capacity * a.row_bytes;
        keys = a.cache + base;
        values = a.cache + a.cache_plane + base;
    }
    key_begin = __builtin_amdgcn_readfirstlane(key_begin);
    key_end = __builtin_amdgcn_readfirstlane(key_end);
    row0 = __builtin_amdgcn_readfirstlane(row0);
    const uint64_t line0 = (static_cast<uint64_t>(slot) * a.kv_heads + kv_head) * a.rows;
    if (key_begin >= key_end) {
        // an empty segment: the join takes no more of it than its maximum
        const uint32_t i = row0 + threadIdx.x;
        if (threadIdx.x < 16 && i < row_end) a.partial_ml[line0 + i] = make_float2(neg_inf(), 0.0f);
        return;
    }
    const uint32_t head_off = static_cast<uint32_t>(head_offset<FMT>(kv_head, a.head_dim));
    keys += head_off;
    values += head_off;

    for (uint32_t i = wave; i < NB; i += kAttnWaves) {
        const uint32_t at = min(row0 + n, row_end - 1);
        float x[8];
        load_query8<FMT>(a.q + (static_cast<uint64_t>(at / a.group) * a.q_heads + kv_head * a.group + at % a.group) * a.head_dim,
                         KeyRun<FMT, NB>::unit(quarter, i), a.head_dim, a.scale, x);
        room.queries[2 * i][lane] = f32x4{x[0], x[1], x[2], x[3]};
        room.queries[2 * i + 1][lane] = f32x4{x[4], x[5], x[6], x[7]};
    }
    uint32_t seen = key_end;  // keys below it are seen by the lane's row
    const uint32_t row = row0 + n;
    if (!shared) {
        const uint32_t behind = a.tokens - 1 - (min(row, row_end - 1) - seq * a.seq_rows) / a.group;
        seen = min(length > behind ? length - behind : 0u, key_end);
    }
    if (row >= row_end) seen = 0;
    float m = neg_inf(), l = 0.0f;
    f32x4 out[NG * 4];
#pragma unroll
    for (int i = 0; i < NG * 4; ++i) out[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    KeyRun<FMT, NB> k;
    ValueRun<FMT, NG> raw_v[4];
    const auto rows_of = [&](const uint8_t* plane, uint32_t first) {
        const uint32_t there = first < key_end ? min(key_end - first, 16u) : 0u;
        return TileRows<FMT>(plane, there ? first : key_end - 1, there, a.row_bytes, head_off);
    };
    // offsets are found anew for every tile: kept, they send other numbers to memory
    const auto load_k = [&](uint32_t first) {
        const TileRows<FMT> rows = rows_of(keys, first);
        uint32_t lane4 = quarter;
        asm volatile("" : "+v"(lane4));
        k.load(rows, n, lane4, a.head_dim);
    };
    const auto load_v = [&](uint32_t first) {
        const TileRows<FMT> rows = rows_of(values, first);
        uint32_t lane16 = n;
        asm volatile("" : "+v"(lane16));
#pragma unroll
        for (int r = 0; r < 4; ++r) raw_v[r].load(rows, 4 * quarter + r, lane16, a.head_dim);
    };
    const uint32_t first = key_begin + wave * 16;
    if (first < key_end) {
        load_k(first);
        load_v(first);
    }
    __syncthreads();

    for (uint32_t key0 = first; key0 < key_end; key0 += kAttnWaves * 16) {
        f32x4 s[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float x[8];
            k.values(b, quarter, a.head_dim, key0 + n < key_end, x);
            const f32x4 q0 = room.queries[2 * b][lane], q1 = room.queries[2 * b + 1][lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], q0[j], s[0], 0, 0, 0);
                s[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[4 + j], q1[j], s[1], 0, 0, 0);
            }
            // or every query read is moved up here and the loads in flight to memory
            if (b % 2) __builtin_amdgcn_sched_barrier(0);
        }
        const uint32_t next = key0 + kAttnWaves * 16;
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        float v[4][NG * 4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float x[4];
                raw_v[r].values(g, n, a.head_dim, key0 + 4 * quarter + r < key_end, x);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[r][4 * g + j] = x[j];
            }
        // keys that some rows see and others do not: a value there that is no
        // number must not reach the others as 0 * v
        bool stained = false;
        if (!shared && a.tokens > 1 && key0 + 16 + a.tokens > length + 1) {
            float any = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < NG * 4; ++i) any = __builtin_fmaf(v[r][i], 0.0f, any);
            stained = __builtin_amdgcn_ballot_w64(any != 0.0f) != 0;
        }
        float p[4];
        float top = neg_inf();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            p[r] = key0 + 4 * quarter + r < seen ? s[0][r] + s[1][r] : neg_inf();
            top = fmaxf(top, p[r]);
        }
        if (!shared && a.scores && row < row_end && key0 + 4 * quarter < key_end) {
            const uint64_t line = (static_cast<uint64_t>(seq) * a.kv_heads + kv_head) * a.seq_rows + row - seq * a.seq_rows;
            *reinterpret_cast<f32x4*>(a.scores + line * a.score_pitch + key0 + 4 * quarter) = f32x4{p[0], p[1], p[2], p[3]};
        }
        top = max_xor32(max_xor16(top));
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
            const float m_new = fmaxf(m, top);
            const float fade = m == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= fade;
#pragma unroll
            for (int i = 0; i < NG * 4; ++i) out[i] *= fade;
        }
        const float base = m == neg_inf() ? 0.0f : m;
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(p[r] - base);
        // One rounding of the long sums for every 16 keys, not one a key: with keys
        // alike they all fall to one side (40001 keys a segment 1.4e-4).
        l += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
        for (int block = 0; block < NG * 4; block += kAtOnce) {
            f32x4 sixteen[kAtOnce] = {};
            if (stained) {
                add_seen<NG>(v, p, block, key0, seen, sixteen);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)
                        sixteen[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][block + i], p[r], sixteen[i], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) out[block + i] += sixteen[i];
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(next);
    }

    // join the wavefronts; by way of LDS whole rows are written
    l = sum_xor32(sum_xor16(l));
    __syncthreads();
    if (quarter == 0) room_ml[wave][n] = make_float2(m, l);
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            put_quad<FMT>(room.sums[wave][n], ValueRun<FMT, NG>::quad(4 * quarter + i, g),
                          f32x4{out[4 * g][i], out[4 * g + 1][i], out[4 * g + 2][i], out[4 * g + 3][i]});
    __syncthreads();
    constexpr uint32_t kQuads = kDims / 4;
#pragma unroll
    for (uint32_t i = threadIdx.x; i < 16 * kQuads; i += kAttnThreads) {
        const uint32_t r = i / kQuads, quad = i % kQuads;
        if (row0 + r >= row_end || 4 * quad >= a.head_dim) continue;
        float top = neg_inf(), sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, room_ml[w][r].x);
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) {
            const float2 ml = room_ml[w][r];
            const float f = ml.x == neg_inf() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);
            sum += f * ml.y;
            o += f * *reinterpret_cast<const f32x4*>(&room.sums[w][r][4 * quad]);
        }
        const uint64_t at = line0 + row0 + r;
        if (quad == 0) a.partial_ml[at] = make_float2(top, sum);
        *reinterpret_cast<f32x4*>(a.partial_out + at * a.head_dim + 4 * quad) = o;
    }
}

// One workgroup a row, or 4 LANES dims of one: its segments joined, and for the
// weights its maximum and 1 / sum (0 where it saw nothing), apart: beside a large
// maximum the sum's logarithm has few bits (three equal keys with scores of 2^10
// had weights of 0.33337).
// LANES lanes hold a segment's dims; as many segments as fit the workgroup are
// taken at once, and their sums meet in LDS in the segments' order.  Bound by
// the segments' bytes: 2048 rows of 256 dims with 17 of them 10 us, 3.6 TB/s.
template <int LANES>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(AttnParams a, float* output, float2* shares) {
    constexpr uint32_t kGroups = kAttnThreads / LANES;
    __shared__ float wave_top[kAttnWaves];
    __shared__ f32x4 sums[kGroups][LANES];
    __shared__ float group_l[kGroups];
    const uint64_t all = static_cast<uint64_t>(a.rows) * a.kv_heads;
    const uint64_t row = blockIdx.x;
    const uint32_t slots = a.prefix_slots + a.own_slots;
    const float2* ml = a.partial_ml + row;
    float top = neg_inf();
    for (uint32_t s = threadIdx.x; s < slots; s += kAttnThreads) top = fmaxf(top, ml[s * all].x);
    top = wave_max_tree_f32(top);
    if (threadIdx.x % kWave == 0) wave_top[threadIdx.x / kWave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
    const float base = top == neg_inf() ? 0.0f : top;
    const uint32_t group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const uint32_t dim = 4 * (blockIdx.y * LANES + lane);
    const bool holds = dim < a.head_dim;
    const float* parts = a.partial_out + row * a.head_dim + (holds ? dim : 0);
    // in 64 bits: a cache of 2^29 positions has 65536 segments
    double all_l = 0.0, all_o[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (uint32_t s = group; s < slots; s += kGroups) {
        const float2 x = ml[s * all];
        const f32x4 part = *reinterpret_cast<const f32x4*>(parts + s * all * a.head_dim);
        const float f = __builtin_amdgcn_exp2f(x.x - base);
        all_l += static_cast<double>(f * x.y);
        // an empty segment has left what was there
#pragma unroll
        for (int j = 0; j < 4; ++j) all_o[j] += static_cast<double>(x.x == neg_inf() ? 0.0f : f * part[j]);
    }
    sums[group][lane] = f32x4{static_cast<float>(all_o[0]), static_cast<float>(all_o[1]), static_cast<float>(all_o[2]),
                              static_cast<float>(all_o[3])};
    if (lane == 0) group_l[group] = static_cast<float>(all_l);
    __syncthreads();
    if (group) return;
    float sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t g = 0; g < kGroups; ++g) {
        sum += group_l[g];
        o += sums[g][lane];
    }
    const uint32_t kv_head = static_cast<uint32_t>(row / a.rows), r = static_cast<uint32_t>(row % a.rows);
    if (holds) {
        f32x4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = sum == 0.0f ? 0.0f : o[j] / sum;
        float* p = output + (static_cast<uint64_t>(r / a.group) * a.q_heads + kv_head * a.group + r % a.group) * a.head_dim;
        *reinterpret_cast<f32x4*>(p + dim) = y;
    }
    if (shares && dim == 0) {
        const uint64_t seq = r / a.seq_rows;
        shares[(seq * a.kv_heads + kv_head) * a.seq_rows + r % a.seq_rows] = make_float2(base, sum == 0.0f ? 0.0f : 1.0f / sum);
    }
}

// A lane a position: the weight it got from every row of its sequence.  A
// workgroup's wavefronts take a quarter of the rows each, in row order, and
// their sums meet in order (64 sequences of up to 8192 positions and 8 rows: 9 us).
__global__ __launch_bounds__(kAttnThreads) void attn_weights_kernel(AttnParams a, const float2* shares, const float* in,
                                                                    float* out) {
    __shared__ float sums[kAttnWaves][kWave];
    const uint32_t lane = threadIdx.x % kWave;
    // known to be one for the wavefront, so that its rows' shares are scalar loads
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    const uint32_t key = blockIdx.x * kWave + lane;
    const uint32_t lines = a.kv_heads * a.seq_rows, part = (lines + kAttnWaves - 1) / kAttnWaves;
    const uint32_t begin = min(wave * part, lines), end = min(begin + part, lines);
    // launches have at most 65535 workgroups in y
    for (uint32_t seq = blockIdx.y; seq < a.rows / a.seq_rows; seq += gridDim.y) {
        const uint32_t length = min(a.lengths[seq], a.capacity);
        if (blockIdx.x * kWave >= length) continue;
        const float2* share = shares + static_cast<uint64_t>(seq) * lines;
        const float* scores = a.scores + static_cast<uint64_t>(seq) * lines * a.score_pitch + min(key, length - 1);
        // what an addition rounds off goes into the next: a sequence has up to 2^23
        // rows, whose shares may all round to one side (131072 of them 8.0e-5)
        float sum = 0.0f, lost = 0.0f;
        for (uint32_t i0 = begin; i0 < end; i0 += 4) {
            // four rows' loads on their way, of the last row again where there are fewer
            float x[4];
            float2 of[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t line = min(i0 + i, end - 1);
                x[i] = scores[static_cast<uint64_t>(line) * a.score_pitch];
                of[i] = share[line];
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) x[i] = i0 + i < end ? __builtin_amdgcn_exp2f(x[i] - of[i].x) * of[i].y : 0.0f;
            const float four = ((x[0] + x[1]) + (x[2] + x[3])) - lost, next = sum + four;
            lost = (next - sum) - four;
            sum = next;
        }
        sums[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && key < length) {
            sum = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
            const uint64_t at = static_cast<uint64_t>(seq) * a.capacity + key;
            out[at] = in ? in[at] + sum : sum;
        }
        __syncthreads();
    }
}

// How the work is laid out, and what of the workspace it takes.
struct AttnPlan {
    bool wide;           // the prompt goes by f16 pieces, not with the own rows
    uint32_t prefix_tiles, prefix_slots, own_tiles, own_slots;
    uint64_t out_bytes, ml_bytes, score_bytes, share_bytes, packed_bytes;
    uint32_t score_pitch;
    uint64_t total() const { return out_bytes + ml_bytes + score_bytes + share_bytes + packed_bytes; }
};

uint64_t round256(uint64_t v) { return (v + 255) / 256 * 256; }

// Keys of a segment of attn_rows_kernel: 128 roundings of a wavefront's sums.
constexpr uint32_t kMostRowKeys = 8192;

// Segments of `keys` keys for each of `units` workgroups: `want`, or more where a
// segment's sums would be longer than `longest` keys; `most` at most, and no more
// than a launch holds (2^22 workgroups of 512 threads).
uint32_t segments(uint64_t want, uint32_t keys, uint32_t longest, uint32_t most, uint64_t units) {
    const uint64_t least = (keys + longest - 1) / longest, launch = units < 1u << 22 ? (1u << 22) / units : 1;
    uint64_t n = want < least ? least : want;
    n = n < launch ? n : launch;
    return static_cast<uint32_t>(n < most ? n : most);
}

AttnPlan attn_plan(const PrefixAttentionArgs& s) {
    AttnPlan p{};
    const uint32_t seq_rows = s.tokens * (s.q_heads / s.kv_heads);
    const uint64_t rows = static_cast<uint64_t>(s.sequences) * seq_rows;
    // Workgroups that the chip holds: three to a CU up to 128 dims (five or four
    // fit, and take 0 to 20 % longer), above them two of quantised rows (64 x 4096
    // Q4_0 141 -> 115 us) and one of f32 (two spill: 147 -> 268).  More parts cost
    // their starts and their joins, fewer leave CUs idle.  Own rows of f32 256 x 512,
    // 64 x 8192 (256 dims), Q4_0 24 x 1024 with 5 drafts (128), us:
    //   256  40 / 147 / 34    512  47 / 143 / 31    768  51 / 148 / 28
    //   1024  61 / 143 / 30
    // One sequence behind 100003 rows of 256: 153 us with 32 parts, 87 with 64, 48
    // with 256.
    const uint32_t wanted = s.head_dim <= 128 ? 768 : (s.format == kKvF32 ? 256 : 512);
    uint32_t own_wanted = wanted;
    if (s.prefix_length && rows > 16) {
        p.wide = true;
        const uint32_t pad = s.head_dim <= 64 ? 64 : (s.head_dim <= 128 ? 128 : 256);
        const uint32_t tile = 32 * 256 / pad;
        const uint32_t most = (s.prefix_length + tile - 1) / tile;
        // Packing converts a tile of keys once, not once for every 64 rows, for a
        // launch and a copy of the tiles: it pays from eight such row tiles and
        // twelve tiles of keys a workgroup on.  Whole calls without and with it, us,
        // rows x prompt, a KV head of 256 dims, four of 128, three of 64:
        //   512 x 1000   32 / 39   29 / 37   20 / 24    512 x 4097  39 / 43   43 / 46   31 / 36
        //   1024 x 4097  46 / 48   72 / 66   48 / 46    2048 x 4097 60 / 61  (64 dims) 78 / 67
        //   256 x 32768  61 / 75  100 / 103  68 / 75    512 x 32768 90 / 94  (64 dims) 121 / 97
        // Tiles take as much as the prompt in f32, of which a caller may have none to
        // spare beside a very long one: 4 GiB at most.
        const uint64_t row_tiles = (rows + 63) / 64, packed_bytes = attn_packed_bytes(s.head_dim, s.kv_heads, s.prefix_length);
        const bool packed = row_tiles >= 8 && row_tiles * most * s.kv_heads >= 12 * 256 && packed_bytes <= 1ull << 32;
        if (packed) p.packed_bytes = round256(packed_bytes);
        p.prefix_tiles = static_cast<uint32_t>(packed ? (rows + 127) / 128 : row_tiles);
        const uint64_t units = static_cast<uint64_t>(p.prefix_tiles) * s.kv_heads;
        const uint64_t want = units >= 256 ? 1 : 256 / units;  // one workgroup to a CU
        p.prefix_slots = segments(want, s.prefix_length, kMostPromptKeys, most, units);
    } else if (s.prefix_length) {
        p.prefix_tiles = static_cast<uint32_t>((rows + 15) / 16);
        const uint64_t units = static_cast<uint64_t>(p.prefix_tiles) * s.kv_heads;
        const uint32_t most = (s.prefix_length + 63) / 64;
        // one launch for both: shared by their lengths, so that all of it is at work at once
        const uint32_t mine = static_cast<uint32_t>(static_cast<uint64_t>(wanted) * s.prefix_length / (static_cast<uint64_t>(s.prefix_length) + s.capacity));
        own_wanted = wanted - mine;
        p.prefix_slots = segments(mine < units ? 1 : mine / units, s.prefix_length, kMostRowKeys, most, units);
    }
    if (s.capacity) {
        p.own_tiles = (seq_rows + 15) / 16;
        const uint64_t units = static_cast<uint64_t>(p.own_tiles) * s.kv_heads * s.sequences;
        const uint32_t most = (s.capacity + 63) / 64;
        const uint64_t want = own_wanted < units ? 1 : (own_wanted + units - 1) / units;
        p.own_slots = segments(want, s.capacity, kMostRowKeys, most, units);
    }
    const uint64_t lines = rows * s.kv_heads, parts = lines * (p.prefix_slots + p.own_slots);
    p.out_bytes = round256(parts * s.head_dim * 4);
    p.ml_bytes = round256(parts * 8);
    if (s.weights_out) {
        p.score_pitch = (s.capacity + 3) / 4 * 4;
        p.score_bytes = round256(lines * p.score_pitch * 4);
        p.share_bytes = round256(lines * sizeof(float2));
    }
    return p;
}

template <int FMT, int NB>
void launch_rows(hipStream_t stream, uint32_t items, const AttnParams& a) {
    hipLaunchKernelGGL((attn_rows_kernel<FMT, NB>), dim3(items), dim3(kAttnThreads), 0, stream, a);
}

template <int FMT>
void launch_rows(hipStream_t stream, uint32_t items, const AttnParams& a) {
    if (a.head_dim <= 64)
        launch_rows<FMT, 2>(stream, items, a);
    else if (a.head_dim <= 128)
        launch_rows<FMT, 4>(stream, items, a);
    else
        launch_rows<FMT, 8>(stream, items, a);
}

}  // namespace

uint64_t prefix_attention_workspace(const PrefixAttentionArgs& s) { return attn_plan(s).total(); }

hipError_t launch_prefix_attention(hipStream_t stream, const PrefixAttentionArgs& s) {
    const AttnPlan p = attn_plan(s);
    uint8_t* ws = static_cast<uint8_t*>(s.workspace);
    AttnParams a{};
    a.q = s.q;
    a.prefix = s.prefix;
    a.cache = s.cache;
    a.lengths = s.lengths;
    a.partial_out = reinterpret_cast<float*>(ws);
    a.partial_ml = reinterpret_cast<float2*>(ws + p.out_bytes);
    a.scores = s.weights_out ? reinterpret_cast<float*>(ws + p.out_bytes + p.ml_bytes) : nullptr;
    float2* shares = s.weights_out ? reinterpret_cast<float2*>(ws + p.out_bytes + p.ml_bytes + p.score_bytes) : nullptr;
    const uint32_t width = s.kv_heads * s.head_dim;
    a.row_bytes = s.format == kKvF32 ? width * 4 : width / 32 * (s.format == kKvQ8_0 ? 34 : 18);
    a.prefix_plane = static_cast<uint64_t>(s.prefix_capacity) * a.row_bytes;
    a.cache_plane = static_cast<uint64_t>(s.sequences) * s.capacity * a.row_bytes;
    a.prefix_length = s.prefix_length;
    a.capacity = s.capacity;
    a.score_pitch = p.score_pitch;
    a.tokens = s.tokens;
    a.q_heads = s.q_heads;
    a.kv_heads = s.kv_heads;
    a.group = s.q_heads / s.kv_heads;
    a.head_dim = s.head_dim;
    a.seq_rows = s.tokens * a.group;
    a.rows = s.sequences * a.seq_rows;
    a.prefix_tiles = p.prefix_tiles;
    a.prefix_slots = p.prefix_slots;
    a.own_tiles = p.own_tiles;
    a.own_slots = p.own_slots;
    a.scale = s.scale * kLog2e;
    const uint32_t prefix_items = p.prefix_tiles * p.prefix_slots * s.kv_heads;
    if (!p.wide) a.prefix_items = prefix_items;
    const uint32_t items = a.prefix_items + s.sequences * s.kv_heads * p.own_slots * p.own_tiles;
    hipError_t e = hipSuccess;
    void* packed = p.packed_bytes ? ws + p.out_bytes + p.ml_bytes + p.score_bytes + p.share_bytes : nullptr;
    if (p.wide && (e = launch_attn_wide(stream, s.format, prefix_items, a, packed)) != hipSuccess) return e;
    if (items) {
        if (s.format == kKvF32)
            launch_rows<kKvF32>(stream, items, a);
        else if (s.format == kKvQ8_0)
            launch_rows<kKvQ8_0>(stream, items, a);
        else
            launch_rows<kKvQ4_0>(stream, items, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const uint64_t all = static_cast<uint64_t>(a.rows) * a.kv_heads;
    // Few rows have many segments, and a workgroup for every 64 dims of one reads
    // them sooner: 64 rows of 256 with 520 segments 18.9 -> 8.6 us.
    const uint32_t pieces = all < 512 ? (s.head_dim + 63) / 64 : 1;
    const dim3 join_grid(static_cast<uint32_t>(all), pieces), join_block(kAttnThreads);
    if (s.head_dim <= 64 * pieces)
        hipLaunchKernelGGL(attn_join_kernel<16>, join_grid, join_block, 0, stream, a, s.output, shares);
    else if (s.head_dim <= 128)
        hipLaunchKernelGGL(attn_join_kernel<32>, join_grid, join_block, 0, stream, a, s.output, shares);
    else
        hipLaunchKernelGGL(attn_join_kernel<64>, join_grid, join_block, 0, stream, a, s.output, shares);
    e = hipGetLastError();
    if (e != hipSuccess || !s.weights_out) return e;
    hipLaunchKernelGGL(attn_weights_kernel, dim3((s.capacity + kWave - 1) / kWave, s.sequences < 65535 ? s.sequences : 65535),
                       dim3(kAttnThreads), 0, stream, a, shares, s.weights_in, s.weights_out);
    return hipGetLastError();
}

}  // namespace atlas
