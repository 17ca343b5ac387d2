// paged_attention_kernels.hip -- attention over a cache in pages: how the work
// is split, and the join of rows that were.  No counterpart in the reference,
// whose executors decode one sequence from a contiguous cache.
#include "paged_attention.hpp"

namespace atlas {
namespace {

// One workgroup a query row, or 4 LANES dims of one: its parts joined, where
// there is more than one, or zero where nothing was seen.  LANES lanes hold a
// part's dims; as many parts as fit the workgroup are taken at once, and their
// sums meet in the wavefront and then in LDS, in an order of their own.  The loads' latency is its time: a
// group's first parts are on their way before the row's maximum is known.
template <int LANES, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_join_kernel(PagedAttnParams a) {
    constexpr uint32_t kGroups = THREADS / LANES, kWaves = THREADS / kWave, kAtOnce = 4;
    __shared__ float wave_top[kWaves];
    __shared__ f32x4 sums[kWaves][LANES];
    __shared__ float wave_l[kWaves];
    const uint32_t seq = blockIdx.x / a.q_heads, q_head = blockIdx.x % a.q_heads;
    const uint32_t kv_head = q_head / a.group, in_group = q_head % a.group;
    const PagedRow row = a.rows[(static_cast<uint64_t>(seq) * a.kv_heads + kv_head) * a.head_tiles + in_group / kPagedHeads];
    const SeenRange seen = seen_of(a, seq);
    const uint32_t group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const uint32_t dim = 4 * (blockIdx.y * LANES + lane);
    const bool holds = dim < a.head_dim;
    float* out = a.output + static_cast<uint64_t>(blockIdx.x) * a.head_dim + dim;
    if (seen.hi == seen.lo) {  // no part has the row
        if (group == 0 && holds) *reinterpret_cast<f32x4*>(out) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        return;
    }
    if (row.first == row.last) return;
    const uint32_t count = row.last - row.first + 1, head = in_group % kPagedHeads;
    // a row begins in the second slot of its first part and goes on in the others' first
    const auto line_of = [&](uint32_t i) { return (2ull * (row.first + i) + (i == 0 ? 1 : 0)) * a.heads + head; };
    float2 ml[kAtOnce];
    f32x4 part[kAtOnce];
    const auto load = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j) {
            const uint64_t line = line_of(min(i0 + j * kGroups, count - 1));
            ml[j] = a.partial_ml[line];
            part[j] = *reinterpret_cast<const f32x4*>(a.partial_out + line * a.head_dim + (holds ? dim : 0));
        }
    };
    load(group);
    float top = neg_inf();
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) top = fmaxf(top, a.partial_ml[line_of(i)].x);
    top = wave_max_tree_f32(top);
    if (threadIdx.x % kWave == 0) wave_top[threadIdx.x / kWave] = top;
    __syncthreads();
    top = wave_top[0];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) top = fmaxf(top, wave_top[w]);
    const float base = top == neg_inf() ? 0.0f : top;
    // in 64 bits: a row has up to 2^20 parts
    double all_l = 0.0, all_o[4] = {0.0, 0.0, 0.0, 0.0};
    for (uint32_t i0 = group; i0 < count; i0 += kAtOnce * kGroups) {
        if (i0 != group) load(i0);
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j) {
            const float f = i0 + j * kGroups < count ? __builtin_amdgcn_exp2f(ml[j].x - base) : 0.0f;
            all_l += static_cast<double>(f * ml[j].y);
#pragma unroll
            for (int k = 0; k < 4; ++k) all_o[k] += static_cast<double>(f * part[j][k]);
        }
    }
    // the groups of a wavefront, then the wavefronts
    const auto join = [&](double all) {
        float x = static_cast<float>(all);
        if constexpr (LANES <= 8) x += dpp_f32<0x128, 0xf, false>(x);  // row_ror:8
        if constexpr (LANES <= 16) x = sum_xor16(x);
        if constexpr (LANES <= 32) x = sum_xor32(x);
        return x;
    };
    const f32x4 mine = {join(all_o[0]), join(all_o[1]), join(all_o[2]), join(all_o[3])};
    const float mine_l = join(all_l);
    if (threadIdx.x % kWave < LANES) sums[threadIdx.x / kWave][lane] = mine;
    if (threadIdx.x % kWave == 0) wave_l[threadIdx.x / kWave] = mine_l;
    __syncthreads();
    if (group || !holds) return;
    float sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) {
        sum += wave_l[i];
        o += sums[i][lane];
    }
    f32x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = sum == 0.0f ? 0.0f : o[j] / sum;
    *reinterpret_cast<f32x4*>(out) = y;
}

constexpr uint32_t kJoinThreads = 256;

// Additions to a wavefront's sums in a part, a unit each: with keys alike they all round to
// one side, 2^-25 of the sum at most each.
constexpr uint32_t kPartUnits = 256 * kPagedAttnWaves;
constexpr uint32_t kMostParts = 1u << 20;

uint64_t round256(uint64_t v) { return (v + 255) / 256 * 256; }

struct PagedPlan {
    uint32_t few_parts, most_parts, heads;
    uint64_t out_bytes, ml_bytes, row_bytes;
};

PagedPlan paged_plan(const PagedCache& c, uint32_t q_heads) {
    PagedPlan p{};
    const uint32_t group = q_heads / c.kv_heads;
    p.heads = group < kPagedHeads ? group : kPagedHeads;
    const uint32_t unit = paged_keys(c.format);
    const uint64_t capacity = static_cast<uint64_t>(c.table_width) * c.page_size;
    const uint64_t rows = static_cast<uint64_t>(c.sequences) * c.kv_heads * ((group + kPagedHeads - 1) / kPagedHeads);
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
uint32_t whole_row_units(const PagedCache& c, uint32_t window, uint64_t rows) {
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

}  // namespace

uint64_t paged_attention_workspace(const PagedCache& c, uint32_t q_heads) {
    const PagedPlan p = paged_plan(c, q_heads);
    return p.out_bytes + p.ml_bytes + p.row_bytes;
}

hipError_t launch_paged_attention(hipStream_t stream, const PagedAttentionArgs& s) {
    const PagedCache& c = s.cache;
    const PagedPlan p = paged_plan(c, s.q_heads);
    PagedAttnParams a{};
    a.q = s.q;
    a.pages = c.pages;
    a.table = c.table;
    a.lengths = s.lengths;
    a.output = s.output;
    a.partial_out = static_cast<float*>(s.workspace);
    a.partial_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(s.workspace) + p.out_bytes);
    a.rows = reinterpret_cast<PagedRow*>(static_cast<uint8_t*>(s.workspace) + p.out_bytes + p.ml_bytes);
    a.page_bytes = paged_page_bytes(c);
    a.part_bytes = paged_part_bytes(c.format, c.page_size, c.head_dim);
    a.page_count = c.page_count;
    a.page_shift = static_cast<uint32_t>(__builtin_ctz(c.page_size));
    a.table_width = c.table_width;
    a.sequences = c.sequences;
    a.capacity = c.table_width * c.page_size;
    a.kv_heads = c.kv_heads;
    a.group = s.q_heads / c.kv_heads;
    a.head_tiles = (a.group + kPagedHeads - 1) / kPagedHeads;
    a.heads = p.heads;
    a.q_heads = s.q_heads;
    a.head_dim = c.head_dim;
    a.window = s.window;
    a.few_parts = p.few_parts;
    a.most_parts = p.most_parts;
    a.part_units = kPartUnits;
    a.row_units = whole_row_units(c, s.window, c.sequences * c.kv_heads * a.head_tiles);
    a.scale = s.scale * kLog2e;
    hipError_t e;
    switch (c.format) {
        case kKvF32: e = launch_paged_attention_f32(stream, a); break;
        case kKvF16: e = launch_paged_attention_f16(stream, a); break;
        case kKvQ8_0: e = launch_paged_attention_q8_0(stream, a); break;
        default: e = launch_paged_attention_q4_0(stream, a); break;
    }
    if (e != hipSuccess || a.row_units) return e;
    const uint32_t lines = c.sequences * s.q_heads;
    // Few rows have many parts: a workgroup for every 64 dims of one, and of 16 wavefronts; for every 32 where they
    // have 128 and more (8 heads of 256 dims, 512 parts 34.1 us for 35.0; 32 parts the other way, 13.5 for 13.9).
    if (lines < 64 && p.most_parts / (c.sequences * c.kv_heads * a.head_tiles) >= 128) {
        hipLaunchKernelGGL((paged_join_kernel<8, 1024>), dim3(lines, (c.head_dim + 31) / 32), dim3(1024), 0, stream, a);
        return hipGetLastError();
    }
    if (lines < 512) {
        hipLaunchKernelGGL((paged_join_kernel<16, 1024>), dim3(lines, (c.head_dim + 63) / 64), dim3(1024), 0, stream, a);
        return hipGetLastError();
    }
    const dim3 grid(lines), block(kJoinThreads);
    if (c.head_dim <= 64)
        hipLaunchKernelGGL((paged_join_kernel<16, kJoinThreads>), grid, block, 0, stream, a);
    else if (c.head_dim <= 128)
        hipLaunchKernelGGL((paged_join_kernel<32, kJoinThreads>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((paged_join_kernel<64, kJoinThreads>), grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace atlas
