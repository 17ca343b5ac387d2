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
// 32 is eight lanes and a wavefront holds 64 / LANES rows.  A rotating lane loads
// its partners' dims too: the line is there, and nothing is exchanged.  Bound by
// bytes, and below a few hundred tokens by the chain of its loads (position,
// table, store).
#include "device_common.hpp"
#include "paged_layout.hpp"

namespace atlas {
namespace {

constexpr uint32_t kPagedThreads = 256;
constexpr uint32_t kPagedWaves = kPagedThreads / kWave;
constexpr uint32_t kNoPlace = 0xffffffffu;

typedef f32x4 f32x4_row __attribute__((aligned(4)));

struct Place {
    uint32_t page, row;  // page kNoPlace: the position has none
};

__device__ __forceinline__ Place place_of(const PagedCache& c, uint32_t shift, uint32_t sequence, uint32_t position) {
    const uint32_t entry = position >> shift;
    if (sequence >= c.sequences || entry >= c.table_width) return {kNoPlace, 0};
    const uint32_t page = c.table[static_cast<uint64_t>(sequence) * c.table_width + entry];
    return {page < c.page_count ? page : kNoPlace, position & (c.page_size - 1)};
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

template <int FMT, int LANES>
__global__ __launch_bounds__(kPagedThreads) void paged_append_kernel(PagedAppendArgs a, uint32_t shift) {
    constexpr uint32_t kRows = kWave / LANES;  // of a wavefront
    const PagedCache& c = a.cache;
    const uint32_t hd = c.head_dim, heads = a.query ? a.q_heads : 0, each = heads + 2 * c.kv_heads;
    const uint64_t row = (static_cast<uint64_t>(blockIdx.x) * kPagedWaves + threadIdx.x / kWave) * kRows + threadIdx.x % kWave / LANES;
    const uint32_t token = static_cast<uint32_t>(row / each);
    const uint32_t head = static_cast<uint32_t>(row % each);  // queries, keys, values
    if (token >= a.tokens) return;
    const uint32_t dim = threadIdx.x % LANES * 4;
    const bool holds = dim < hd;
    const uint32_t sequence = a.sequences ? a.sequences[token] : token, position = a.positions[token];
    if (sequence >= c.sequences || position >> shift >= c.table_width) return;
    const bool is_query = head < heads, is_key = !is_query && head < heads + c.kv_heads;
    const uint32_t kv_head = is_query ? 0 : (head - heads) % c.kv_heads;
    const float* in = is_query ? a.query + (static_cast<uint64_t>(token) * heads + head) * hd
                               : (is_key ? a.key : a.value) + (static_cast<uint64_t>(token) * c.kv_heads + kv_head) * hd;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (holds) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(in + dim);
        if ((is_query || is_key) && a.cosine) {
            const uint32_t half = hd / 2;
            const float* cosine = a.cosine + static_cast<uint64_t>(position) * a.rope_stride;
            const float* sine = a.sine + static_cast<uint64_t>(position) * a.rope_stride;
            f32x4 y, cs, sn;  // the partners; the lane's angles
            if (half % 4 == 0) {
                const uint32_t at = dim < half ? dim : dim - half;
                y = *reinterpret_cast<const f32x4*>(in + (dim < half ? dim + half : at));
                cs = *reinterpret_cast<const f32x4_row*>(cosine + at);
                sn = *reinterpret_cast<const f32x4_row*>(sine + at);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t d = dim + j, at = d < half ? d : d - half;
                    y[j] = in[d < half ? d + half : at];
                    cs[j] = cosine[at];
                    sn[j] = sine[at];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float turned = y[j] * sn[j], kept = x[j] * cs[j];
                v[j] = dim + j < half ? kept - turned : turned + kept;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = x[j];
        }
    }
    if (is_query) {
        // query_out may be query: the row has been read by its wavefront, whose stores follow
        if (holds)
            *reinterpret_cast<f32x4*>(a.query_out + (static_cast<uint64_t>(token) * heads + head) * hd + dim) =
                f32x4{v[0], v[1], v[2], v[3]};
        return;
    }
    const Place at = place_of(c, shift, sequence, position);
    if (at.page == kNoPlace) return;
    uint8_t* part = part_of_page(c, at.page, is_key ? 0 : 1, kv_head, paged_part_bytes(FMT, c.page_size, hd));
    const uint32_t row_bytes = paged_row_code_bytes(FMT, hd);
    uint8_t* to = part + at.row * row_bytes;
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
        if (is_key) {
            if constexpr (FMT == kKvQ8_0)
                *reinterpret_cast<uint32_t*>(to + dim) = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
            else
                *reinterpret_cast<uint16_t*>(to + dim / 2) =
                    static_cast<uint16_t>(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const uint32_t place = paged_value_place(hd, dim + j);
                if constexpr (FMT == kKvQ8_0)
                    *reinterpret_cast<uint16_t*>(to + place) = static_cast<uint16_t>(code[j] | code[j + 1] << 8);
                else
                    to[place / 2] = static_cast<uint8_t>(code[j] | code[j + 1] << 4);
            }
        }
        if (threadIdx.x % 8 == 0)
            *reinterpret_cast<uint16_t*>(part + c.page_size * row_bytes +
                                         2 * ((at.row / 4 * (hd / 32) + dim / 32) * 4 + at.row % 4)) = f2h(scale);
    }
}

// Bound by what it writes, 4 bytes a value.
template <int FMT, int LANES>
__global__ __launch_bounds__(kPagedThreads) void paged_read_kernel(PagedReadArgs a, uint32_t shift) {
    constexpr uint32_t kRows = kWave / LANES;
    const PagedCache& c = a.cache;
    const uint32_t hd = c.head_dim, each = 2 * c.kv_heads;
    const uint64_t row = (static_cast<uint64_t>(blockIdx.x) * kPagedWaves + threadIdx.x / kWave) * kRows + threadIdx.x % kWave / LANES;
    const uint32_t token = static_cast<uint32_t>(row / each);
    const uint32_t head = static_cast<uint32_t>(row % each);  // keys, values
    const uint32_t dim = threadIdx.x % LANES * 4;
    if (token >= a.rows || dim >= hd) return;
    const uint32_t plane = head / c.kv_heads, kv_head = head % c.kv_heads;
    float* out = plane ? a.value : a.key;
    if (!out) return;
    const Place at = place_of(c, shift, a.sequences ? a.sequences[token] : token, a.positions[token]);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (at.page != kNoPlace) {
        const uint8_t* part = part_of_page(c, at.page, plane, kv_head, paged_part_bytes(FMT, c.page_size, hd));
        const uint32_t row_bytes = paged_row_code_bytes(FMT, hd);
        const uint8_t* from = part + at.row * row_bytes;
        if constexpr (FMT == kKvF32) {
            v = *reinterpret_cast<const f32x4*>(from + 4 * dim);
        } else if constexpr (FMT == kKvF16) {
            const u32x2_t w = *reinterpret_cast<const u32x2_t*>(from + 2 * dim);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = h2f(static_cast<uint16_t>(w[j / 2] >> (16 * (j % 2))));
        } else {
            const float scale = h2f(*reinterpret_cast<const uint16_t*>(
                part + c.page_size * row_bytes + 2 * ((at.row / 4 * (hd / 32) + dim / 32) * 4 + at.row % 4)));
            uint32_t w;
            if (plane == 0) {
                w = FMT == kKvQ8_0 ? *reinterpret_cast<const uint32_t*>(from + dim) : *reinterpret_cast<const uint16_t*>(from + dim / 2);
            } else {
                const uint32_t p0 = paged_value_place(hd, dim), p1 = paged_value_place(hd, dim + 2);
                w = FMT == kKvQ8_0 ? *reinterpret_cast<const uint16_t*>(from + p0) |
                                         static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(from + p1)) << 16
                                   : from[p0 / 2] | static_cast<uint32_t>(from[p1 / 2]) << 8;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float code = FMT == kKvQ8_0 ? static_cast<float>(static_cast<int8_t>(w >> (8 * j)))
                                                  : static_cast<float>(w >> (4 * j) & 15u) - 8.0f;
                v[j] = code * scale;
            }
        }
    }
    *reinterpret_cast<f32x4*>(out + (static_cast<uint64_t>(token) * c.kv_heads + kv_head) * hd + dim) = v;
}

uint32_t shift_of(uint32_t page_size) { return static_cast<uint32_t>(__builtin_ctz(page_size)); }

template <int LANES>
uint32_t groups_for(uint64_t rows) {
    constexpr uint32_t kEach = kPagedThreads / LANES;
    return static_cast<uint32_t>((rows + kEach - 1) / kEach);
}

template <int FMT, int LANES>
hipError_t launch_append(hipStream_t stream, const PagedAppendArgs& a) {
    const uint64_t rows = static_cast<uint64_t>(a.tokens) * ((a.query ? a.q_heads : 0) + 2 * a.cache.kv_heads);
    hipLaunchKernelGGL((paged_append_kernel<FMT, LANES>), dim3(groups_for<LANES>(rows)), dim3(kPagedThreads), 0, stream, a,
                       shift_of(a.cache.page_size));
    return hipGetLastError();
}
template <int FMT, int LANES>
hipError_t launch_read(hipStream_t stream, const PagedReadArgs& a) {
    const uint64_t rows = static_cast<uint64_t>(a.rows) * 2 * a.cache.kv_heads;
    hipLaunchKernelGGL((paged_read_kernel<FMT, LANES>), dim3(groups_for<LANES>(rows)), dim3(kPagedThreads), 0, stream, a,
                       shift_of(a.cache.page_size));
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
