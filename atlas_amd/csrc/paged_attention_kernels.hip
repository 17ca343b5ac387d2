// paged_attention_kernels.hip -- attention over a cache in pages: its launches,
// and the join of rows that were split.  No counterpart in the reference, whose
// executors decode one sequence from a contiguous cache.
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
    const uint32_t last_part = a.most_parts - 1;
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
    // of a length that changed between the launches whatever lies there: no other parts than there are
    const uint32_t first = min(row.first, last_part);
    const uint32_t count = min(row.last - row.first, last_part - first) + 1, head = in_group % kPagedHeads;
    // a row begins in the second slot of its first part and goes on in the others' first
    const auto line_of = [&](uint32_t i) { return (2ull * (first + i) + (i == 0 ? 1 : 0)) * a.heads + head; };
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

}  // namespace

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
    a.head_tiles = paged_head_tiles(c, s.q_heads);
    a.heads = p.heads;
    a.q_heads = s.q_heads;
    a.head_dim = c.head_dim;
    a.window = s.window;
    a.few_parts = p.few_parts;
    a.most_parts = p.most_parts;
    a.part_units = kPartUnits;
    a.row_units = whole_row_units(c, s.window, paged_rows(c, s.q_heads));
    a.scale = s.scale * kLog2e;
    hipError_t e;
    switch (c.format) {
        case kKvF32: e = launch_paged_attention_f32(stream, a); break;
        case kKvF16: e = launch_paged_attention_f16(stream, a); break;
        case kKvQ8_0: e = launch_paged_attention_q8_0(stream, a); break;
        default: e = launch_paged_attention_q4_0(stream, a); break;
    }
    if (e != hipSuccess || a.row_units) return e;
    const PagedJoin j = paged_join(c, s.q_heads, p.most_parts);
    const dim3 grid(c.sequences * s.q_heads, j.groups), block(j.threads);
    if (j.lanes == 8)
        hipLaunchKernelGGL((paged_join_kernel<8, kFewThreads>), grid, block, 0, stream, a);
    else if (j.threads == kFewThreads)
        hipLaunchKernelGGL((paged_join_kernel<16, kFewThreads>), grid, block, 0, stream, a);
    else if (j.lanes == 16)
        hipLaunchKernelGGL((paged_join_kernel<16, kJoinThreads>), grid, block, 0, stream, a);
    else if (j.lanes == 32)
        hipLaunchKernelGGL((paged_join_kernel<32, kJoinThreads>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((paged_join_kernel<64, kJoinThreads>), grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace atlas
