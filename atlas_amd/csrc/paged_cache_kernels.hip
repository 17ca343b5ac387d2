// paged_cache_kernels.hip -- keys and values into the pages of a cache, with
// the rotation to their positions, and back out of them as f32.  No counterpart
// in the reference, whose caches are contiguous; the rotation is its half-split
// RoPE (crates/atlas-metal/src/kernels.metal:940-994) and the Q8_0 / Q4_0
// encoders those of its KV append (:1197-1267), on the blocks of a head.
//
// Append, of token t at position p of its sequence:
//   x'_i         = x_i c_i - x_{i + h} s_i,   i < h = head_dim / 2
//   x'_{i + h}   = x_i s_i + x_{i + h} c_i,   c, s the tables' row p
// for every head of its key and query; key and value go to row p % page_size of
// page table[sequence, p / page_size], the query to query_out.  Products and sums
// are rounded one by one, as everywhere here.
//
// A row (a head's query, key or value) is LANES lanes of four dims, so a block of
// 32 is eight lanes, and a wavefront holds 64 / LANES rows at once, all of one
// token: where the token goes is known to the wavefront by scalar loads, and a
// lane's angles serve all of its rows.  A rotating lane loads its partners' dims
// too: the line is there, and nothing is exchanged.  Bound by bytes (4096 tokens of
// 32 + 8 heads of 128 dims to f16 31 to 33 us, 5.7 TB/s read and written, to Q8_0 and Q4_0
// 34, 5.2), and below a
// few hundred tokens by the chain of its loads (position, table, store): 3 to 5 us.
#include "device_common.hpp"
#include "paged_layout.hpp"

namespace atlas {
namespace {

constexpr uint32_t kPagedThreads = 256;
constexpr uint32_t kPagedWaves = kPagedThreads / kWave;

typedef f32x4 f32x4_row __attribute__((aligned(4)));

// Where a token's rows are: known to the whole wavefront.
struct Place {
    uint32_t page, row;
    bool in_range, there;  // the position is one of the table's; it has a page
};

__device__ __forceinline__ Place place_of(const PagedCache& c, uint32_t shift, uint32_t sequence, uint32_t position) {
    const uint32_t entry = position >> shift;
    Place p{0, position & (c.page_size - 1), sequence < c.sequences && entry < c.table_width, false};
    if (p.in_range) {
        p.page = c.table[static_cast<uint64_t>(sequence) * c.table_width + entry];
        p.there = p.page < c.page_count;
    }
    return p;
}

// A wavefront's token and its share of the token's rows, 2^chunks shares.
struct Share {
    uint32_t token, first;
};
__device__ __forceinline__ Share share_of(uint32_t chunks, uint32_t steps) {
    const uint32_t wave = blockIdx.x * kPagedWaves + static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    return {wave >> chunks, (wave & ((1u << chunks) - 1)) * steps};
}
constexpr int kAtOnce = 4;  // rows of a lane on their way

// f32 rows for whoever comes next: past the caches where there are more of them than
// the L2s hold (4096 tokens of 32 heads 40.3 -> 32.5 us), into them where not.
constexpr uint64_t kCachedBytes = 32u << 20;
template <bool PAST>
__device__ __forceinline__ void put_f32(float* to, f32x4 v) {
    if constexpr (PAST)  // at run time the two are taken for one, a plain one
        __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(to));
    else
        *reinterpret_cast<f32x4*>(to) = v;
}

// The codes of a row, four to a lane, from the order of the dims to a value's or
// back: through LDS, so that memory sees whole rows (two loads of two codes a lane
// keep the address unit busy for as long as the rows of 32768 positions take, 83 us).
// A wavefront's room has a word for every lane of every step.
typedef uint32_t CodeRoom[kAtOnce][kWave];
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ uint8_t* part_of_page(const PagedCache& c, uint32_t page, uint32_t plane, uint32_t head, uint32_t part_bytes) {
    return c.pages + (static_cast<uint64_t>(page) * 2 * c.kv_heads + plane * c.kv_heads + head) * part_bytes;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}
// Over the eight lanes of a block: xor 1, xor 2, then the other four mirrored.
__device__ __forceinline__ float block_max(float v) {
    v = fmaxf(v, dpp_f32<0xb1, 0xf, false>(v));
    v = fmaxf(v, dpp_f32<0x4e, 0xf, false>(v));
    return fmaxf(v, dpp_f32<0x141, 0xf, false>(v));
}
__device__ __forceinline__ uint32_t block_min(uint32_t v) {
    v = min(v, dpp_u32<0xb1>(v));
    v = min(v, dpp_u32<0x4e>(v));
    return min(v, dpp_u32<0x141>(v));
}

// The codes of a lane's four values and their block's scale, as the KV append
// encodes them.
template <int FMT>
__device__ __forceinline__ void encode(const float (&v)[4], uint32_t (&code)[4], float& scale) {
    const float amax = block_max(fmaxf(fmaxf(fmaxf(0.0f, __builtin_fabsf(v[0])), __builtin_fabsf(v[1])),
                                       fmaxf(__builtin_fabsf(v[2]), __builtin_fabsf(v[3]))));
    if (FMT == kKvQ8_0) {
        scale = amax == 0.0f ? 0.0f : fdiv_rn(amax, 127.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = fminf(fmaxf(fdiv_rn(v[j], scale), -127.0f), 127.0f);
            code[j] = scale == 0.0f ? 0u : static_cast<uint32_t>(static_cast<int>(roundf(x))) & 255u;
        }
    } else {
        // the sign of the first value as large as any
        uint32_t first = 64;
#pragma unroll
        for (int j = 3; j >= 0; --j)
            if (__builtin_fabsf(v[j]) == amax) first = (threadIdx.x % 8 * 4 + j) * 2 + (__float_as_uint(v[j]) >> 31);
        first = block_min(first);
        scale = amax == 0.0f ? 0.0f : fdiv_rn(first & 1 ? -amax : amax, -8.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float t = fdiv_rn(v[j], scale) + 8.5f;
            code[j] = scale == 0.0f ? 0u : t >= 15.0f ? 15u : t > 0.0f ? static_cast<uint32_t>(t) : 0u;
        }
    }
}

// One head's row of four dims a lane, stored: `to` is the page's part.
template <int FMT>
__device__ __forceinline__ void store_row(uint8_t* part, const PagedCache& c, uint32_t row, uint32_t dim, bool is_key, bool holds,
                                          uint32_t p0, uint32_t p1, uint8_t* room, const float (&v)[4]) {
    const uint32_t hd = c.head_dim, row_bytes = paged_row_code_bytes(FMT, hd);
    uint8_t* to = part + row * row_bytes;
    if constexpr (FMT == kKvF32) {
        if (holds) *reinterpret_cast<f32x4*>(to + 4 * dim) = f32x4{v[0], v[1], v[2], v[3]};
    } else if constexpr (FMT == kKvF16) {
        if (holds)
            *reinterpret_cast<u32x2_t*>(to + 2 * dim) =
                u32x2_t{f2h(v[0]) | static_cast<uint32_t>(f2h(v[1])) << 16, f2h(v[2]) | static_cast<uint32_t>(f2h(v[3])) << 16};
    } else {
        uint32_t code[4];
        float scale;
        encode<FMT>(v, code, scale);
        if (!holds) return;  // head_dim is a multiple of 32: whole blocks
        const uint32_t q0 = is_key ? dim : p0, q1 = is_key ? dim + 2 : p1;
        if constexpr (FMT == kKvQ8_0) {
            *reinterpret_cast<uint16_t*>(room + q0) = static_cast<uint16_t>(code[0] | code[1] << 8);
            *reinterpret_cast<uint16_t*>(room + q1) = static_cast<uint16_t>(code[2] | code[3] << 8);
            wave_lds_fence();
            *reinterpret_cast<uint32_t*>(to + dim) = *reinterpret_cast<const uint32_t*>(room + dim);
        } else {
            room[q0 / 2] = static_cast<uint8_t>(code[0] | code[1] << 4);
            room[q1 / 2] = static_cast<uint8_t>(code[2] | code[3] << 4);
            wave_lds_fence();
            *reinterpret_cast<uint16_t*>(to + dim / 2) = *reinterpret_cast<const uint16_t*>(room + dim / 2);
        }
        if (threadIdx.x % 8 == 0)
            *reinterpret_cast<uint16_t*>(part + c.page_size * row_bytes + 2 * ((row / 4 * (hd / 32) + dim / 32) * 4 + row % 4)) =
                f2h(scale);
    }
}

template <int FMT, int LANES, bool PAST>
__global__ __launch_bounds__(kPagedThreads) void paged_append_kernel(PagedAppendArgs a, uint32_t shift, uint32_t chunks, uint32_t steps) {
    constexpr uint32_t kRows = kWave / LANES;  // of a wavefront at once
    const PagedCache& c = a.cache;
    const uint32_t hd = c.head_dim, half = hd / 2, heads = a.query ? a.q_heads : 0, each = heads + 2 * c.kv_heads;
    const Share share = share_of(chunks, steps);
    if (share.token >= a.tokens) return;
    const uint32_t sequence = a.sequences ? a.sequences[share.token] : share.token, position = a.positions[share.token];
    const Place at = place_of(c, shift, sequence, position);
    if (!at.in_range) return;
    const uint32_t dim = threadIdx.x % LANES * 4;
    const bool holds = dim < hd, turns = a.cosine != nullptr, whole = half % 4 == 0;
    const uint32_t at_dim = holds ? dim : 0, partner = at_dim < half ? at_dim + half : at_dim - half;
    f32x4 cs = {1.0f, 1.0f, 1.0f, 1.0f}, sn = {0.0f, 0.0f, 0.0f, 0.0f};  // the lane's angles
    if (turns) {
        const float* cosine = a.cosine + static_cast<uint64_t>(position) * a.rope_stride;
        const float* sine = a.sine + static_cast<uint64_t>(position) * a.rope_stride;
        if (whole) {
            cs = *reinterpret_cast<const f32x4_row*>(cosine + (at_dim < half ? at_dim : partner));
            sn = *reinterpret_cast<const f32x4_row*>(sine + (at_dim < half ? at_dim : partner));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t d = at_dim + j, i = d < half ? d : d - half;
                cs[j] = cosine[i];
                sn[j] = sine[i];
            }
        }
    }
    const uint32_t part_bytes = paged_part_bytes(FMT, c.page_size, hd);
    __shared__ CodeRoom rooms[paged_quantised(FMT) ? kPagedWaves : 1];
    const uint32_t p0 = paged_quantised(FMT) ? paged_value_place(hd, at_dim) : 0, p1 = paged_quantised(FMT) ? paged_value_place(hd, at_dim + 2) : 0;
    for (uint32_t s0 = 0; s0 < steps; s0 += kAtOnce) {
        f32x4 x[kAtOnce], y[kAtOnce];  // the lane's dims and their partners
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s) {
            if (s0 + s >= steps) break;
            const uint32_t row = min((share.first + s0 + s) * kRows + threadIdx.x % kWave / LANES, each - 1);
            const float* in = row < heads ? a.query + (static_cast<uint64_t>(share.token) * heads + row) * hd
                                          : (row < heads + c.kv_heads ? a.key : a.value) +
                                                (static_cast<uint64_t>(share.token) * c.kv_heads + (row - heads) % c.kv_heads) * hd;
            x[s] = *reinterpret_cast<const f32x4*>(in + at_dim);
            if (!turns) {
                y[s] = x[s];
            } else if (whole) {
                y[s] = *reinterpret_cast<const f32x4*>(in + partner);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) y[s][j] = in[at_dim + j < half ? at_dim + j + half : at_dim + j - half];
            }
        }
        // query_out may be query: a row has been read by its wavefront, and is no other's
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s) {
            const uint32_t row = (share.first + s0 + s) * kRows + threadIdx.x % kWave / LANES;
            if (s0 + s >= steps) break;
            if (row >= each) continue;
            const bool is_query = row < heads, is_key = !is_query && row < heads + c.kv_heads;
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float turned = y[s][j] * sn[j], kept = x[s][j] * cs[j];
                v[j] = !turns || !(is_query || is_key) ? x[s][j] : (dim + j < half ? kept - turned : turned + kept);
                if (!holds) v[j] = 0.0f;
            }
            if (is_query) {
                if (holds)
                    put_f32<PAST>(a.query_out + (static_cast<uint64_t>(share.token) * heads + row) * hd + dim,
                                  f32x4{v[0], v[1], v[2], v[3]});
            } else if (at.there) {
                store_row<FMT>(part_of_page(c, at.page, is_key ? 0 : 1, (row - heads) % c.kv_heads, part_bytes), c, at.row, dim, is_key,
                               holds, p0, p1, reinterpret_cast<uint8_t*>(rooms[paged_quantised(FMT) ? threadIdx.x / kWave : 0][s]) +
                                                  threadIdx.x % kWave / LANES * LANES * 4, v);
            }
        }
    }
}

// The rows that are asked for: of one output that is null neither is read.
__host__ __device__ inline uint32_t read_begin(const PagedReadArgs& a) { return a.key ? 0 : a.cache.kv_heads; }
__host__ __device__ inline uint32_t read_end(const PagedReadArgs& a) { return a.value ? 2 * a.cache.kv_heads : a.cache.kv_heads; }

// Bound by what it writes, 4 bytes a value: 32768 rows of 8 heads of 128 dims from
// Q4_0 48 us, 6.3 TB/s.
template <int FMT, int LANES, bool PAST>
__global__ __launch_bounds__(kPagedThreads) void paged_read_kernel(PagedReadArgs a, uint32_t shift, uint32_t chunks, uint32_t steps) {
    constexpr uint32_t kRows = kWave / LANES;
    const PagedCache& c = a.cache;
    const uint32_t hd = c.head_dim, begin = read_begin(a), end = read_end(a);  // of a token's rows, keys and then values
    const Share share = share_of(chunks, steps);
    if (share.token >= a.rows) return;
    const Place at = place_of(c, shift, a.sequences ? a.sequences[share.token] : share.token, a.positions[share.token]);
    const uint32_t dim = threadIdx.x % LANES * 4;
    if (dim >= hd) return;
    const uint32_t part_bytes = paged_part_bytes(FMT, c.page_size, hd), row_bytes = paged_row_code_bytes(FMT, hd);
    const uint32_t p0 = paged_quantised(FMT) ? paged_value_place(hd, dim) : 0, p1 = paged_quantised(FMT) ? paged_value_place(hd, dim + 2) : 0;
    __shared__ CodeRoom rooms[paged_quantised(FMT) ? kPagedWaves : 1];
    const uint32_t scale_at = c.page_size * row_bytes + 2 * ((at.row / 4 * (hd / 32) + dim / 32) * 4 + at.row % 4);
    for (uint32_t s0 = 0; s0 < steps; s0 += kAtOnce) {
        u32x4_t w[kAtOnce];
        uint32_t scale[kAtOnce];
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s) {
            const uint32_t row = min(begin + (share.first + s0 + s) * kRows + threadIdx.x % kWave / LANES, end - 1);
            const uint32_t plane = row < c.kv_heads ? 0 : 1;
            w[s] = u32x4_t{0, 0, 0, 0};
            scale[s] = 0;
            if (!at.there || s0 + s >= steps) continue;
            const uint8_t* part = part_of_page(c, at.page, plane, row - plane * c.kv_heads, part_bytes);
            const uint8_t* from = part + at.row * row_bytes;
            if constexpr (FMT == kKvF32) {
                w[s] = *reinterpret_cast<const u32x4_t*>(from + 4 * dim);
            } else if constexpr (FMT == kKvF16) {
                const u32x2_t x = *reinterpret_cast<const u32x2_t*>(from + 2 * dim);
                w[s][0] = x[0];
                w[s][1] = x[1];
            } else {
                scale[s] = *reinterpret_cast<const uint16_t*>(part + scale_at);
                w[s][0] = FMT == kKvQ8_0 ? *reinterpret_cast<const uint32_t*>(from + dim) : *reinterpret_cast<const uint16_t*>(from + dim / 2);
            }
        }
        if constexpr (paged_quantised(FMT)) {
#pragma unroll
            for (int s = 0; s < kAtOnce; ++s) {
                const uint32_t row = begin + (share.first + s0 + s) * kRows + threadIdx.x % kWave / LANES;
                uint8_t* codes = reinterpret_cast<uint8_t*>(rooms[threadIdx.x / kWave][s]) + threadIdx.x % kWave / LANES * LANES * 4;
                // a key's four codes lie together, a value's two by two
                const uint32_t q0 = row < c.kv_heads ? dim : p0, q1 = row < c.kv_heads ? dim + 2 : p1;
                if constexpr (FMT == kKvQ8_0) {
                    *reinterpret_cast<uint32_t*>(codes + dim) = w[s][0];
                    wave_lds_fence();
                    w[s][0] = *reinterpret_cast<const uint16_t*>(codes + q0);
                    w[s][1] = *reinterpret_cast<const uint16_t*>(codes + q1);
                } else {
                    *reinterpret_cast<uint16_t*>(codes + dim / 2) = static_cast<uint16_t>(w[s][0]);
                    wave_lds_fence();
                    w[s][0] = codes[q0 / 2];
                    w[s][1] = codes[q1 / 2];
                }
            }
        }
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s) {
            const uint32_t row = begin + (share.first + s0 + s) * kRows + threadIdx.x % kWave / LANES;
            if (s0 + s >= steps || row >= end) continue;
            const uint32_t plane = row < c.kv_heads ? 0 : 1;
            float* out = plane ? a.value : a.key;
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (FMT == kKvF32) {
                    v[j] = __uint_as_float(w[s][j]);
                } else if constexpr (FMT == kKvF16) {
                    v[j] = h2f(static_cast<uint16_t>(w[s][j / 2] >> (16 * (j % 2))));
                } else {
                    const uint32_t two = w[s][j / 2];
                    const float code = FMT == kKvQ8_0 ? static_cast<float>(static_cast<int8_t>(two >> (8 * (j % 2))))
                                                      : static_cast<float>(two >> (4 * (j % 2)) & 15u) - 8.0f;
                    v[j] = code * h2f(static_cast<uint16_t>(scale[s]));
                }
                if (paged_quantised(FMT) && !at.there) v[j] = 0.0f;  // not -0
            }
            put_f32<PAST>(out + (static_cast<uint64_t>(share.token) * c.kv_heads + (row - plane * c.kv_heads)) * hd + dim, v);
        }
    }
}

uint32_t shift_of(uint32_t page_size) { return static_cast<uint32_t>(__builtin_ctz(page_size)); }

// How a token's rows are shared out: few tokens go to many wavefronts, for their
// loads' latency, and many have eight rows a lane, whose loads overlap.
struct Shares {
    uint32_t chunks, steps, groups;
    Shares(uint64_t tokens, uint32_t rows, uint32_t at_once) {
        const uint32_t all = (rows + at_once - 1) / at_once;  // steps of a token
        chunks = 0;
        while ((1u << chunks) < all && (((all + (1u << chunks) - 1) >> chunks) > 8 || tokens << chunks < 4096)) ++chunks;
        steps = (all + (1u << chunks) - 1) >> chunks;
        groups = static_cast<uint32_t>(((tokens << chunks) + kPagedWaves - 1) / kPagedWaves);
    }
};

template <int FMT, int LANES>
hipError_t launch_append(hipStream_t stream, const PagedAppendArgs& a) {
    const Shares s(a.tokens, (a.query ? a.q_heads : 0) + 2 * a.cache.kv_heads, kWave / LANES);
    const bool past = 4ull * a.tokens * a.q_heads * a.cache.head_dim > kCachedBytes;
    const auto kernel = past ? paged_append_kernel<FMT, LANES, true> : paged_append_kernel<FMT, LANES, false>;
    hipLaunchKernelGGL(kernel, dim3(s.groups), dim3(kPagedThreads), 0, stream, a, shift_of(a.cache.page_size), s.chunks, s.steps);
    return hipGetLastError();
}
template <int FMT, int LANES>
hipError_t launch_read(hipStream_t stream, const PagedReadArgs& a) {
    const uint32_t each = read_end(a) - read_begin(a);
    const Shares s(a.rows, each, kWave / LANES);
    const bool past = 4ull * a.rows * each * a.cache.head_dim > kCachedBytes;
    const auto kernel = past ? paged_read_kernel<FMT, LANES, true> : paged_read_kernel<FMT, LANES, false>;
    hipLaunchKernelGGL(kernel, dim3(s.groups), dim3(kPagedThreads), 0, stream, a, shift_of(a.cache.page_size), s.chunks, s.steps);
    return hipGetLastError();
}

// The lanes that four dims each need.
#define ATLAS_PAGED_LANES(FMT, LAUNCH)                                        \
    (a.cache.head_dim <= 32    ? LAUNCH<FMT, 8>(stream, a)                    \
     : a.cache.head_dim <= 64  ? LAUNCH<FMT, 16>(stream, a)                   \
     : a.cache.head_dim <= 128 ? LAUNCH<FMT, 32>(stream, a)                   \
                               : LAUNCH<FMT, 64>(stream, a))
#define ATLAS_PAGED_FORMAT(LAUNCH)                                            \
    switch (a.cache.format) {                                                 \
        case kKvF32: return ATLAS_PAGED_LANES(kKvF32, LAUNCH);                \
        case kKvF16: return ATLAS_PAGED_LANES(kKvF16, LAUNCH);                \
        case kKvQ8_0: return ATLAS_PAGED_LANES(kKvQ8_0, LAUNCH);              \
        default: return ATLAS_PAGED_LANES(kKvQ4_0, LAUNCH);                   \
    }

}  // namespace

hipError_t launch_paged_append(hipStream_t stream, const PagedAppendArgs& a) { ATLAS_PAGED_FORMAT(launch_append) }
hipError_t launch_paged_read(hipStream_t stream, const PagedReadArgs& a) { ATLAS_PAGED_FORMAT(launch_read) }

}  // namespace atlas
