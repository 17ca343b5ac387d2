// logprobs_kernels.hip -- log probabilities of given tokens, entropies and the
// likeliest tokens of rows of logits.  No counterpart in the reference, which
// decodes greedily.
//
// With y_i = (x_i - top) / temperature, top the row's largest logit:
//   S = sum_i e^{y_i},  log p_i = y_i - log S,
//   entropy = -sum_i p_i log p_i = log S + sum_i e^{y_i} (-y_i) / S,
// where every term is positive: nothing cancels.  Probabilities and sums are in
// 64 bits, so a likely token's small log probability keeps its digits.  NaN and
// -inf logits have no mass; all of a row's mass lies on its +inf.
//
// Launches: a wavefront a slice of 1024 logits leaves the slice's sums and the
// maxima of its cells, 128 logits each; one workgroup a row joins them.  The
// likeliest tokens cost the first launch nothing: of 64 groups of cells the k-th
// largest maximum is a border that k tokens reach, so only cells that reach it are
// read again (a few hundred of 2048) and what reaches it in them is ranked.
#include "exp2_f64.hpp"
#include "launch.hpp"

#include <algorithm>
#include <limits>

namespace atlas {
namespace {

constexpr int kLogThreads = 256;
constexpr int kLogWaves = kLogThreads / kWave;
constexpr uint32_t kSlice = 1024;  // a wavefront's, 16 logits a lane
constexpr int kEach = kSlice / kWave;
constexpr uint32_t kCells = 8;     // of a slice: the logits of eight lanes
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr uint32_t kCellList = 1024, kTokenList = 512;

typedef f32x4 f32x4_row __attribute__((aligned(4)));

// Sums of e^{y} and of e^{y} (-y), relative to the slice's top; the cells' maxima.
struct SliceSums {
    double sum, spread;
    float cells[kCells];
};

struct LogprobParams {
    TokenLogprobsArgs s;
    double scale;      // 32 inv_temperature log2(e)
    SliceSums* slices; // [row][slices]
    uint32_t count, blocks;  // slices of a row; workgroups of kLogWaves slices
};

__device__ __forceinline__ float about(float x, float top) {
    return top == __builtin_inff() ? (x == top ? 0.0f : -__builtin_inff()) : x;
}
__device__ __forceinline__ double finite(float top) { return __builtin_isinf(top) ? 0.0 : static_cast<double>(top); }

// Logit i of a lane's, four at a time; lanes 8 r .. 8 r + 7 have cell r.
__device__ __forceinline__ uint32_t slice_at(uint32_t lane, int i) { return (i / 4 * kWave + lane) * 4 + i % 4; }

__device__ __forceinline__ void load_lane(const float* logits, uint32_t first, uint32_t lane, uint32_t vocab, float (&x)[kEach]) {
    if (first + kSlice <= vocab) {
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
            const f32x4 y = *reinterpret_cast<const f32x4_row*>(logits + first + slice_at(lane, 4 * i));
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = number_or_none(y[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t at = first + slice_at(lane, i);
            x[i] = at < vocab ? number_or_none(logits[at]) : -__builtin_inff();
        }
    }
}

template <bool SPREAD>
__global__ __launch_bounds__(kLogThreads) void logprob_sums_kernel(LogprobParams v) {
    __shared__ uint2 table[32];
    const uint32_t row = blockIdx.x / v.blocks, lane = threadIdx.x % kWave;
    const uint32_t slice = blockIdx.x % v.blocks * kLogWaves + threadIdx.x / kWave;
    float x[kEach];
    load_lane(v.s.logits + row * v.s.row_stride, min(slice, v.count - 1) * kSlice, lane, v.s.vocab, x);
    Exp2::fill(table);
    const Exp2 exp2_of(table);
    __syncthreads();
    if (slice >= v.count) return;
    float cell = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kEach; ++i) cell = fmaxf(cell, x[i]);
    cell = fmaxf(cell, dpp_f32<0xb1, 0xf, false>(cell));
    cell = fmaxf(cell, dpp_f32<0x4e, 0xf, false>(cell));
    cell = fmaxf(cell, dpp_f32<0x141, 0xf, false>(cell));
    const float top = wave_max_tree_f32(cell);
    if (top == __builtin_inff()) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) x[i] = about(x[i], top);
    }
    const double zero = finite(top);
    double sum = 0.0, spread = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const double y = fmax((static_cast<double>(x[i]) - zero) * v.scale, exp2_of.least);
        const double e = exp2_of(y);
        sum += e;
        if (SPREAD) spread = __builtin_fma(e, -y, spread);
    }
    sum = wave_sum_f64(sum);
    if (SPREAD) spread = wave_sum_f64(spread);
    SliceSums* out = v.slices + static_cast<uint64_t>(row) * v.count + slice;
    if (lane == 0) {
        out->sum = sum;
        out->spread = spread;
    }
    if (lane % 8 == 0) out->cells[lane / 8] = cell;
}

// A logit's place among all: larger first, of equal ones the lower index; 0: none.
__device__ __forceinline__ uint32_t ordered(float x) {
    x += 0.0f;  // -0 is +0
    const uint32_t u = __float_as_uint(x);
    return x > -__builtin_inff() ? (u >> 31 ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ uint64_t place_of(float x, uint32_t index) {
    const uint32_t u = ordered(x);
    return u ? static_cast<uint64_t>(u) << 32 | static_cast<uint32_t>(~index) : 0u;
}
__device__ __forceinline__ float value_of(uint32_t u) { return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u); }

// Every logit of the cells that reach `border`, by eight lanes a cell.
template <class F>
__device__ __forceinline__ void for_cell(const float* logits, uint32_t cell, uint32_t vocab, F&& f) {
    const uint32_t lane = threadIdx.x % 8 + cell % kCells * 8, first = cell / kCells * kSlice;
    float x[kEach];
    load_lane(logits, first, lane, vocab, x);
#pragma unroll
    for (int i = 0; i < kEach; ++i) f(x[i], first + slice_at(lane, i));
}

// The place that exactly `k` tokens reach, by eight bits a pass over the cells
// that reach `border`: for rows where too many tokens are level for a list.
__device__ uint64_t exact_border(const LogprobParams& v, const float* logits, const SliceSums* slices, uint32_t border, uint32_t k,
                                 uint32_t (&bins)[256], uint64_t& state, uint32_t& left) {
    if (threadIdx.x == 0) {
        state = 0;
        left = k;
    }
    for (int shift = 56; shift >= 0; shift -= 8) {
        bins[threadIdx.x] = 0;
        __syncthreads();
        const uint64_t above = state;
        for (uint32_t cell = threadIdx.x / 8; cell < v.count * kCells; cell += kLogThreads / 8) {
            if (ordered(slices[cell / kCells].cells[cell % kCells]) < border) continue;
            for_cell(logits, cell, v.s.vocab, [&](float x, uint32_t index) {
                const uint64_t place = place_of(x, index);
                if (place && (shift == 56 || place >> (shift + 8) == above >> (shift + 8))) atomicAdd(&bins[place >> shift & 255], 1u);
            });
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t need = left, bin = 256;
            while (bin-- > 0 && bins[bin] < need) need -= bins[bin];
            // fewer than k in all: the first pass ends below its lowest bin, and every token counts
            if (bin == 0xffffffffu) {
                left = 0;
            } else {
                state = above | static_cast<uint64_t>(bin) << shift;
                left = need;
            }
        }
        __syncthreads();
        if (left == 0) return 1;
    }
    return state;
}

// One workgroup a row.
__global__ __launch_bounds__(kLogThreads) void logprob_rows_kernel(LogprobParams v) {
    __shared__ uint2 table[32];
    __shared__ double wave_sum[kLogWaves], wave_spread[kLogWaves];
    __shared__ float wave_top[kLogWaves];
    __shared__ uint32_t border_room, cell_count, token_count, left_room;
    __shared__ uint64_t state_room;
    __shared__ union {
        struct {
            uint32_t cells[kCellList];
            uint64_t tokens[kTokenList];
        } list;
        uint32_t bins[256];
    } room;
    const TokenLogprobsArgs& s = v.s;
    const uint32_t row = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const float* logits = s.logits + row * s.row_stride;
    const SliceSums* slices = v.slices + static_cast<uint64_t>(row) * v.count;
    Exp2::fill(table);
    const Exp2 exp2_of(table);

    // the row's top, and with it the border: the k-th largest of 64 groups' maxima
    const uint32_t cells = v.count * kCells;
    float mine = -__builtin_inff();
    for (uint32_t i = threadIdx.x; i < cells; i += kLogThreads) mine = fmaxf(mine, slices[i / kCells].cells[i % kCells]);
    const float wtop = wave_max_tree_f32(mine);
    if (lane == 0) wave_top[wave] = wtop;
    __shared__ float group_top[kLogThreads];
    group_top[threadIdx.x] = mine;
    if (threadIdx.x == 0) cell_count = token_count = 0;
    __syncthreads();
    const float top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
    if (s.top && wave == 0) {
        uint32_t group = 0;
        for (int w = 0; w < kLogWaves; ++w) group = max(group, ordered(group_top[w * kWave + lane]));
        uint32_t border = 0;
#pragma unroll
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t with = border | 1u << bit;
            if (static_cast<uint32_t>(__builtin_popcountll(__builtin_amdgcn_ballot_w64(group >= with))) >= s.top) border = with;
        }
        if (lane == 0) border_room = max(border, 1u);
    }

    double sum = 0.0, spread = 0.0;
    for (uint32_t i = threadIdx.x; i < v.count; i += kLogThreads) {
        const SliceSums x = slices[i];
        float slice_top = x.cells[0];
#pragma unroll
        for (uint32_t j = 1; j < kCells; ++j) slice_top = fmaxf(slice_top, x.cells[j]);
        const double y = fmax((static_cast<double>(about(slice_top, top)) - finite(top)) * v.scale, exp2_of.least);
        const double f = exp2_of(y);
        sum = __builtin_fma(f, x.sum, sum);
        spread = __builtin_fma(f, __builtin_fma(-y, x.sum, x.spread), spread);
    }
    sum = wave_sum_f64(sum);
    spread = wave_sum_f64(spread);
    if (lane == 0) {
        wave_sum[wave] = sum;
        wave_spread[wave] = spread;
    }
    __syncthreads();
    sum = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
    spread = (wave_spread[0] + wave_spread[1]) + (wave_spread[2] + wave_spread[3]);
    const bool any = top > -__builtin_inff();
    const double log_sum = any ? log(sum) : 0.0;
    const auto logprob = [&](float x) {
        const double y = (static_cast<double>(about(number_or_none(x), top)) - finite(top)) * s.inv_temperature - log_sum;
        return any ? static_cast<float>(y) : -__builtin_inff();
    };
    if (s.entropy && threadIdx.x == 0)
        // thirty-seconds of powers of two to natural units
        s.entropy[row] = any ? static_cast<float>(log_sum + spread / sum * (0x1.62e42fefa39efp-1 / 32.0)) : 0.0f;
    for (uint32_t i = threadIdx.x; i < s.given; i += kLogThreads) {
        const uint64_t at = static_cast<uint64_t>(row) * s.given + i;
        const uint32_t token = s.tokens[at];
        s.logprobs[at] = token < s.vocab ? logprob(logits[token]) : -__builtin_inff();
    }
    if (!s.top) return;

    const uint32_t border = border_room;
    for (uint32_t i = threadIdx.x; i < cells; i += kLogThreads)
        if (ordered(slices[i / kCells].cells[i % kCells]) >= border) {
            const uint32_t at = atomicAdd(&cell_count, 1u);
            if (at < kCellList) room.list.cells[at] = i;
        }
    __syncthreads();
    uint64_t reach = static_cast<uint64_t>(border) << 32;
    const auto push = [&](float x, uint32_t index) {
        const uint64_t place = place_of(x, index);
        if (place >= reach) {
            const uint32_t at = atomicAdd(&token_count, 1u);
            if (at < kTokenList) room.list.tokens[at] = place;
        }
    };
    if (cell_count <= kCellList)
        for (uint32_t i = threadIdx.x / 8; i < cell_count; i += kLogThreads / 8) for_cell(logits, room.list.cells[i], s.vocab, push);
    __syncthreads();
    if (cell_count > kCellList || token_count > kTokenList) {
        __syncthreads();
        if (threadIdx.x == 0) token_count = 0;
        reach = exact_border(v, logits, slices, border, s.top, room.bins, state_room, left_room);
        __syncthreads();
        for (uint32_t i = threadIdx.x / 8; i < cells; i += kLogThreads / 8)
            if (ordered(slices[i / kCells].cells[i % kCells]) >= border) for_cell(logits, i, s.vocab, push);
        __syncthreads();
    }
    const uint32_t count = token_count;
    for (uint32_t i = threadIdx.x; i < count; i += kLogThreads) {
        const uint64_t place = room.list.tokens[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < count; ++j) rank += room.list.tokens[j] > place;
        if (rank < s.top) {
            s.top_ids[static_cast<uint64_t>(row) * s.top + rank] = ~static_cast<uint32_t>(place);
            s.top_logprobs[static_cast<uint64_t>(row) * s.top + rank] = logprob(value_of(static_cast<uint32_t>(place >> 32)));
        }
    }
    for (uint32_t i = count + threadIdx.x; i < s.top; i += kLogThreads) {
        s.top_ids[static_cast<uint64_t>(row) * s.top + i] = kNoToken;
        s.top_logprobs[static_cast<uint64_t>(row) * s.top + i] = -__builtin_inff();
    }
}

uint32_t slices_of(uint32_t vocab) { return (vocab + kSlice - 1) / kSlice; }

}  // namespace

uint64_t token_logprobs_workspace(uint32_t rows, uint32_t vocab, uint32_t) {
    return static_cast<uint64_t>(rows) * slices_of(vocab) * sizeof(SliceSums);
}

hipError_t launch_token_logprobs(hipStream_t stream, const TokenLogprobsArgs& s) {
    LogprobParams v{};
    v.s = s;
    // finite, or the top itself would be 0 times infinity
    v.scale = std::min(32.0 * 1.4426950408889634074 * s.inv_temperature, std::numeric_limits<double>::max());
    v.slices = static_cast<SliceSums*>(s.workspace);
    v.count = slices_of(s.vocab);
    v.blocks = (v.count + kLogWaves - 1) / kLogWaves;
    const dim3 grid(s.rows * v.blocks), block(kLogThreads);
    if (s.entropy)
        hipLaunchKernelGGL(logprob_sums_kernel<true>, grid, block, 0, stream, v);
    else
        hipLaunchKernelGGL(logprob_sums_kernel<false>, grid, block, 0, stream, v);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(logprob_rows_kernel, dim3(s.rows), block, 0, stream, v);
    return hipGetLastError();
}

}  // namespace atlas
