// logprobs_kernels.hip -- log probabilities of given tokens, entropies and the
// likeliest tokens of rows of logits.  No counterpart in the reference, which
// decodes greedily.
//
// With y_i = (x_i - top) / temperature, top the row's largest logit:
//   S = sum_i e^{y_i},  log p_i = y_i - log S,
//   entropy = -sum_i p_i log p_i = log S + sum_i e^{y_i} (-y_i) / S,
// where every term is positive: nothing cancels.  Probabilities and sums are in
// 64 bits, and S is kept as what it has beside the top's own 1: of a likely token
// that is its log probability, which so keeps its digits however small it is.  NaN
// and -inf logits have no mass; all of a row's mass lies on its +inf.
//
// Launches: a wavefront a slice of one or two strips of 1024 logits leaves the slice's sums and the
// maxima of its cells, 128 logits each; one workgroup a row joins them.  The
// likeliest tokens cost the first launch nothing: of 64 or 256 groups of cells the k-th
// largest maximum is a border that k tokens reach, so only cells that reach it are
// read again (some 25 of 2048 for 20 tokens) and what reaches it in them is ranked.
// Bound by the bytes and nearly as much by the 64-bit instructions: 256 rows of 262144
// logits 55 to 56 us in the first launch, 4.8 TB/s (random numbers are read at 5.8 at
// best), and 8.3 in the second; 2048 of 50257 84 to 87 and 7.
#include "exp2_f64.hpp"
#include "logprobs_plan.hpp"

#include <algorithm>
#include <limits>

namespace atlas {
namespace {

constexpr uint32_t kCells = 8;     // of a strip: the logits of eight lanes
constexpr int kEach = kStrip / kWave;
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr uint32_t kCellList = 1024, kTokenList = 512;

// A slice's sums of e^{y}, less its top's own 1, and of e^{y} (-y), relative to its
// top, y in thirty-seconds of powers of two.
struct SliceSums {
    double rest, spread;
};
// Sums that hold a 1 lose what is below its last bit, which matters where there is
// little else: less than this in every lane, the top's apart.  (More of it in the sum,
// and 45 additions move it by 2^-39 at most.)
constexpr double kLittle = 0x1p-8;

struct LogprobParams {
    TokenLogprobsArgs s;
    double scale;            // 32 inv_temperature log2(e)
    SliceSums* slices;       // [row][slices]
    float* cells;            // [row][strips][kCells]: their maxima
    uint32_t strips, count;  // strips and slices of a row
    uint32_t each;           // strips of a slice
};

__device__ __forceinline__ float about(float x, float top) {
    return top == __builtin_inff() ? (x == top ? 0.0f : -__builtin_inff()) : x;
}
__device__ __forceinline__ double finite(float top) { return __builtin_isinf(top) ? 0.0 : static_cast<double>(top); }

// Logit i of a lane's in a strip, four at a time; lanes 8 r .. 8 r + 7 have cell r.
__device__ __forceinline__ uint32_t slice_at(uint32_t lane, int i) { return (i / 4 * kWave + lane) * 4 + i % 4; }

// Behind a row's end a load brings zeros, which are no logits of it.
__device__ __forceinline__ void load_lane(__amdgpu_buffer_rsrc_t logits, uint32_t first, uint32_t lane, float (&x)[kEach]) {
#pragma unroll
    for (int i = 0; i < kEach / 4; ++i) {
        const f32x4 y = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(logits, (first + slice_at(lane, 4 * i)) * 4, 0, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = y[j];
    }
}
__device__ __forceinline__ void end_lane(uint32_t first, uint32_t lane, uint32_t vocab, float (&x)[kEach]) {
    if (first + kStrip > vocab)
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (first + slice_at(lane, i) >= vocab) x[i] = -__builtin_inff();
}

// 2^(y / 256), y <= 0, as Exp2 has 2^(y / 32): of a table of 256 the polynomial needs
// three degrees: of r^4, |r| <= 1 / 2, the second one takes a r^2, which leaves least at
// a = (sqrt 2 - 1) / 2, and the whole within 2^-45.  A table's place is a byte of the
// sum; its bits come along with the exponent, so a table entry has them taken out.
struct FineExp2 {
    static constexpr uint32_t kSize = 256;
    const uint2* table;
    double c[3], shift, least;

    static __device__ void fill(uint2 (&table)[kSize]) {
        static_assert(kSize == kLogThreads);
        const uint32_t i = threadIdx.x;
        const uint64_t bits = __builtin_bit_cast(uint64_t, exp2(i * (1.0 / kSize)));
        table[i] = make_uint2(static_cast<uint32_t>(bits), static_cast<uint32_t>(bits >> 32) - (1023u << 20) - (i << 12));
    }
    explicit __device__ FineExp2(const uint2 (&table)[kSize])
        : table(table),
          c{0x1.c6b08d704a0c0p-5 * 0x1p-24,  // ln2^3 / 6, of 1 / 256 each
            0x1.ebfbe40c8b585p-3 * 0x1p-16,  // ln2^2 / 2 + a ln2^4 / 24 / 256^2
            0x1.62e42fefa39efp-1 * 0x1p-8},  // ln2
          shift(0x1.8p52 + kSize * 1023.0), least(-1022.0 * kSize) {
        asm("" : "+v"(c[0]));
#pragma unroll
        for (int i = 1; i < 3; ++i) asm("" : "+s"(c[i]));
        asm("" : "+s"(shift));
    }
    __device__ __forceinline__ double operator()(double y) const {  // y >= least
        const double t = y + shift;
        const double r = y - (t - shift);
        const uint32_t k = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, t));
        double p = __builtin_fma(c[0], r, c[1]);
        p = __builtin_fma(p, r, c[2]);
        p = __builtin_fma(p, r, 1.0);
        uint2 power = table[k % kSize];
        power.y += k << 12;
        return p * __builtin_bit_cast(double, static_cast<uint64_t>(power.y) << 32 | power.x);
    }
};

// Workgroups that stay: eight to a CU, and the table's filling, behind the first
// logits' loads, once for all of a workgroup's slices.  Bound by the bytes and the
// 64-bit instructions together, so a logit takes as few as there are: one that is no
// number, and one too far below the top to have mass, become in one instruction the
// lowest that has hardly any.
template <bool SPREAD, int STRIPS>
__global__ __launch_bounds__(kLogThreads, 8) void logprob_sums_kernel(LogprobParams v) {
    __shared__ uint2 table[FineExp2::kSize];
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    // a wavefront's slices of all rows', every `step`-th
    const uint64_t items = static_cast<uint64_t>(v.s.rows) * v.count;
    const uint32_t step = gridDim.x * kLogWaves, first = min(blockIdx.x * kLogWaves + wave, static_cast<uint32_t>(items - 1));
    uint32_t row = first / v.count, slice = first % v.count;
    const uint32_t row_step = step / v.count, slice_step = step % v.count;
    float x[STRIPS][kEach];
    const auto load = [&] {
        const auto logits = span_rsrc(v.s.logits + row * v.s.row_stride, v.s.vocab * 4);
#pragma unroll
        for (int i = 0; i < STRIPS; ++i) load_lane(logits, (slice * STRIPS + i) * kStrip, lane, x[i]);
    };
    load();
    FineExp2::fill(table);
    const FineExp2 exp2_of(table);
    const double scale = fmin(v.scale * 8.0, 0x1.fffffffffffffp1023);
    __syncthreads();
    for (uint64_t item = blockIdx.x * kLogWaves + wave; item < items; item += step) {
        const uint64_t at = static_cast<uint64_t>(row) * v.count + slice;
        float cell[STRIPS], most = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < STRIPS; ++i) {
            end_lane((slice * STRIPS + i) * kStrip, lane, v.s.vocab, x[i]);
            cell[i] = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < kEach; ++j) cell[i] = fmaxf(cell[i], x[i][j]);
            cell[i] = fmaxf(cell[i], dpp_f32<0xb1, 0xf, false>(cell[i]));
            cell[i] = fmaxf(cell[i], dpp_f32<0x4e, 0xf, false>(cell[i]));
            cell[i] = fmaxf(cell[i], dpp_f32<0x141, 0xf, false>(cell[i]));
            most = fmaxf(most, cell[i]);
        }
        const float top = wave_max_tree_f32(most);
        const double zero = finite(top);
        double sum = 0.0, spread = 0.0;
        if (top == __builtin_inff())
#pragma unroll
            for (int i = 0; i < STRIPS; ++i)
#pragma unroll
                for (int j = 0; j < kEach; ++j) x[i][j] = about(x[i][j], top);
#pragma unroll
        for (int i = 0; i < STRIPS; ++i)
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const double y = fmax((static_cast<double>(x[i][j]) - zero) * scale, exp2_of.least), e = exp2_of(y);
                sum += e;
                if (SPREAD) spread = __builtin_fma(e, -y, spread);
            }
        // here, and not behind the next logits' loads, beside which these would have to be kept
        asm volatile("" : "+v"(sum), "+v"(spread));
        const bool has_top = sum >= 1.0;
        const bool little = __builtin_popcountll(__builtin_amdgcn_ballot_w64(has_top)) == 1 &&
                            __builtin_amdgcn_ballot_w64((has_top ? sum - 1.0 : sum) > kLittle) == 0;
        if (little) {  // the top's lane again, without it
            double rest = 0.0;
#pragma unroll
            for (int i = 0; i < STRIPS; ++i)
#pragma unroll
                for (int j = 0; j < kEach; ++j) {
                    asm volatile("" : "+v"(x[i][j]), "+v"(rest));  // one by one, and no power kept from above
                    const double y = fmax((static_cast<double>(x[i][j]) - zero) * scale, exp2_of.least), e = exp2_of(y);
                    rest += y == 0.0 ? 0.0 : e;
                }
            asm volatile("" : "+v"(rest));
            if (has_top) sum = rest;
        }
        float* cells = v.cells + static_cast<uint64_t>(row) * v.strips * kCells;
        const uint32_t strip = slice * STRIPS;
        row += row_step;
        slice += slice_step;
        if (slice >= v.count) {
            slice -= v.count;
            ++row;
        }
        if (item + step < items) load();
        sum = wave_sum_f64(sum);
        if (SPREAD) spread = wave_sum_f64(spread);
        if (lane == 0) v.slices[at] = SliceSums{little ? sum : sum - 1.0, spread * (1.0 / 8.0)};
        if (lane % 8 == 0)
#pragma unroll
            for (uint32_t i = 0; i < STRIPS; ++i)
                if (strip + i < v.strips) cells[static_cast<uint64_t>(strip + i) * kCells + lane / 8] = cell[i];
    }
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
    const uint32_t lane = threadIdx.x % 8 + cell % kCells * 8, first = cell / kCells * kStrip;
    float x[kEach];
    load_lane(span_rsrc(logits, vocab * 4), first, lane, x);
    end_lane(first, lane, vocab, x);
#pragma unroll
    for (int i = 0; i < kEach; ++i) f(x[i], first + slice_at(lane, i));
}

// The place that exactly `k` tokens reach, by eight bits a pass over the cells
// that reach `border`: for rows where too many tokens are level for a list.  1
// where there are fewer than k.
template <int THREADS>
__device__ uint64_t exact_border(const LogprobParams& v, const float* logits, const float* cells, uint32_t border, uint32_t k,
                                 uint32_t (&bins)[256], uint64_t& state, uint32_t& left) {
    if (threadIdx.x == 0) {
        state = 0;
        left = k;
    }
    for (int shift = 56; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) bins[threadIdx.x] = 0;
        __syncthreads();
        const uint64_t above = state;
        for (uint32_t cell = threadIdx.x / 8; cell < v.strips * kCells; cell += THREADS / 8) {
            if (ordered(cells[cell]) < border) continue;
            for_cell(logits, cell, v.s.vocab, [&](float x, uint32_t index) {
                const uint64_t place = place_of(x, index);
                if (place && (shift == 56 || place >> (shift + 8) == above >> (shift + 8))) atomicAdd(&bins[place >> shift & 255], 1u);
            });
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t need = left, bin = 256;
            while (bin-- > 0 && bins[bin] < need) need -= bins[bin];
            if (bin == 0xffffffffu) {  // fewer than k in all, known after the first pass
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

// log(1 + r), r >= 0, to 2^-42 of it: where 1 + r would lose more, five terms of its series.
// (The library's log1p takes 0.3 us more of a row.)
__device__ __forceinline__ double log_one_and(double r) {
    if (r >= kLittle) return log(1.0 + r);
    return r * __builtin_fma(r, __builtin_fma(r, __builtin_fma(r, __builtin_fma(r, 1.0 / 5.0, -1.0 / 4.0), 1.0 / 3.0), -1.0 / 2.0), 1.0);
}

// The s.top-th largest of 64 EACH groups' maxima, to 21 bits of its place, by one wavefront.
template <int EACH, int THREADS>
__device__ __forceinline__ uint32_t border_of(const float (&maxima)[THREADS], uint32_t lane, uint32_t k) {
    uint32_t group[EACH];
#pragma unroll
    for (uint32_t j = 0; j < EACH; ++j) {
        float x = -__builtin_inff();
#pragma unroll
        for (uint32_t i = 0; i < THREADS / (EACH * kWave); ++i) x = fmaxf(x, maxima[(i * EACH + j) * kWave + lane]);
        group[j] = ordered(x);
    }
    uint32_t border = 0;
#pragma unroll
    for (uint32_t bit = 1u << 31; bit >= 1u << 11; bit >>= 1) {
        const uint32_t with = border | bit;
        uint32_t reached = 0;
#pragma unroll
        for (uint32_t j = 0; j < EACH; ++j)
            reached += static_cast<uint32_t>(__builtin_popcountll(__builtin_amdgcn_ballot_w64(group[j] >= with)));
        if (reached >= k) border = with;
    }
    return border;
}

// One workgroup a row (row_threads).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void logprob_rows_kernel(LogprobParams v) {
    constexpr uint32_t kWaves = THREADS / kWave;
    __shared__ uint2 table[32];
    __shared__ double wave_rest[kWaves], wave_spread[kWaves];
    __shared__ float wave_top[kWaves], group_top[THREADS];
    __shared__ uint32_t border_room, cell_count, token_count, top_count, left_room;
    __shared__ uint64_t state_room;
    __shared__ union {
        struct {
            uint32_t cells[kCellList];
            uint64_t tokens[kTokenList];
        } list;
        uint32_t bins[256];
    } room;
    const TokenLogprobsArgs& s = v.s;
    const uint32_t row = blockIdx.x, lane = threadIdx.x % kWave;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    const float* logits = s.logits + row * s.row_stride;
    const SliceSums* slices = v.slices + static_cast<uint64_t>(row) * v.count;
    const float* cells = v.cells + static_cast<uint64_t>(row) * v.strips * kCells;
    const uint32_t cells_of_row = v.strips * kCells;
    // the table is filled while the first loads are on their way
    const float first_cell = threadIdx.x < cells_of_row ? cells[threadIdx.x] : -__builtin_inff();
    const uint32_t idle = s.top ? kWave : 0;  // threads that look for the border instead
    SliceSums first_slice{0.0, 0.0};
    if (threadIdx.x >= idle && threadIdx.x - idle < v.count) first_slice = slices[threadIdx.x - idle];
    __builtin_amdgcn_sched_barrier(0);
    Exp2::fill(table);
    const Exp2 exp2_of(table);
    float mine = first_cell;
    for (uint32_t i = threadIdx.x + THREADS; i < cells_of_row; i += THREADS) mine = fmaxf(mine, cells[i]);
    const float wtop = wave_max_tree_f32(mine);
    if (lane == 0) wave_top[wave] = wtop;
    group_top[threadIdx.x] = mine;
    if (threadIdx.x == 0) cell_count = token_count = top_count = 0;
    __syncthreads();
    float top = wave_top[0];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) top = fmaxf(top, wave_top[w]);

    // one wavefront finds the border while the others sum
    const bool finds = s.top && wave == 0;
    double rest = 0.0, spread = 0.0;
    if (finds) {
        // 64 groups do for few tokens: 20 of them leave some 24 above the border
        const uint32_t border = s.top <= 24 ? border_of<1, THREADS>(group_top, lane, s.top) : border_of<4, THREADS>(group_top, lane, s.top);
        if (lane == 0) border_room = max(border, 1u);
    } else {
        for (uint32_t i = threadIdx.x - idle; i < v.count; i += THREADS - idle) {
            const SliceSums x = i + idle < THREADS ? first_slice : slices[i];
            float slice_top = -__builtin_inff();
            // the last slice may have a strip less
            for (uint32_t j = i * v.each * kCells; j < min((i + 1) * v.each * kCells, cells_of_row); j += 4) {
                const f32x4 c = *reinterpret_cast<const f32x4*>(cells + j);
                slice_top = fmaxf(slice_top, fmaxf(fmaxf(c.x, c.y), fmaxf(c.z, c.w)));
            }
            const double y = fmax((static_cast<double>(about(slice_top, top)) - finite(top)) * v.scale, exp2_of.least);
            const double f = exp2_of(y);
            rest = __builtin_fma(f, x.rest, rest);
            if (f == 1.0)
                atomicAdd(&top_count, 1u);  // a slice with the row's top, or as good as it
            else
                rest += f;
            spread = __builtin_fma(f, __builtin_fma(-y, 1.0 + x.rest, x.spread), spread);
        }
        rest = wave_sum_f64(rest);
        spread = wave_sum_f64(spread);
    }
    if (lane == 0) {
        wave_rest[wave] = rest;
        wave_spread[wave] = spread;
    }
    __syncthreads();
    rest = spread = 0.0;
    for (uint32_t w = 0; w < kWaves; ++w) {
        rest += wave_rest[w];
        spread += wave_spread[w];
    }
    rest += static_cast<double>(top_count) - 1.0;
    const bool any = top > -__builtin_inff();
    const double log_sum = any ? log_one_and(rest) : 0.0;
    const auto logprob = [&](float x) {
        const double y = (static_cast<double>(about(number_or_none(x), top)) - finite(top)) * s.inv_temperature - log_sum;
        return any ? static_cast<float>(y) + 0.0f : -__builtin_inff();  // not -0
    };
    if (s.entropy && threadIdx.x == 0)
        // thirty-seconds of powers of two to natural units
        s.entropy[row] = any ? static_cast<float>(log_sum + spread / (1.0 + rest) * (0x1.62e42fefa39efp-1 / 32.0)) : 0.0f;
    for (uint32_t i = threadIdx.x; i < s.given; i += THREADS) {
        const uint64_t at = static_cast<uint64_t>(row) * s.given + i;
        const uint32_t token = s.tokens[at];
        s.logprobs[at] = token < s.vocab ? logprob(logits[token]) : -__builtin_inff();
    }
    if (!s.top) return;

    const uint32_t border = border_room;
    for (uint32_t i = threadIdx.x; i < cells_of_row; i += THREADS)
        if (ordered(i < THREADS ? first_cell : cells[i]) >= border) {
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
        for (uint32_t i = threadIdx.x / 8; i < cell_count; i += THREADS / 8) for_cell(logits, room.list.cells[i], s.vocab, push);
    __syncthreads();
    if (cell_count > kCellList || token_count > kTokenList) {
        __syncthreads();
        if (threadIdx.x == 0) token_count = 0;
        reach = exact_border<THREADS>(v, logits, cells, border, s.top, room.bins, state_room, left_room);
        __syncthreads();
        for (uint32_t i = threadIdx.x / 8; i < cells_of_row; i += THREADS / 8)
            if (ordered(cells[i]) >= border) for_cell(logits, i, s.vocab, push);
        __syncthreads();
    }
    const uint32_t count = token_count;
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
        const uint64_t place = room.list.tokens[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < count; ++j) rank += room.list.tokens[j] > place;
        if (rank < s.top) {
            s.top_ids[static_cast<uint64_t>(row) * s.top + rank] = ~static_cast<uint32_t>(place);
            s.top_logprobs[static_cast<uint64_t>(row) * s.top + rank] = logprob(value_of(static_cast<uint32_t>(place >> 32)));
        }
    }
    for (uint32_t i = count + threadIdx.x; i < s.top; i += THREADS) {
        s.top_ids[static_cast<uint64_t>(row) * s.top + i] = kNoToken;
        s.top_logprobs[static_cast<uint64_t>(row) * s.top + i] = -__builtin_inff();
    }
}

}  // namespace

uint64_t token_logprobs_workspace(uint32_t rows, uint32_t vocab, uint32_t) {
    return static_cast<uint64_t>(rows) * (slices_of(rows, vocab) * sizeof(SliceSums) + strips_of(vocab) * kCells * sizeof(float));
}

hipError_t launch_token_logprobs(hipStream_t stream, const TokenLogprobsArgs& s) {
    LogprobParams v{};
    v.s = s;
    // finite, or the top itself would be 0 times infinity
    v.scale = std::min(32.0 * 1.4426950408889634074 * s.inv_temperature, std::numeric_limits<double>::max());
    v.slices = static_cast<SliceSums*>(s.workspace);
    v.strips = strips_of(s.vocab);
    v.count = slices_of(s.rows, s.vocab);
    v.each = strips_each(s.rows, s.vocab);
    v.cells = reinterpret_cast<float*>(v.slices + static_cast<uint64_t>(s.rows) * v.count);
    const dim3 grid(sum_groups(s.rows, s.vocab)), block(kLogThreads);
    const auto sums = s.entropy ? (v.each == 2 ? logprob_sums_kernel<true, 2> : logprob_sums_kernel<true, 1>)
                                : (v.each == 2 ? logprob_sums_kernel<false, 2> : logprob_sums_kernel<false, 1>);
    hipLaunchKernelGGL(sums, grid, block, 0, stream, v);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (row_threads(s.rows) == 1024)
        hipLaunchKernelGGL(logprob_rows_kernel<1024>, dim3(s.rows), dim3(1024), 0, stream, v);
    else
        hipLaunchKernelGGL(logprob_rows_kernel<256>, dim3(s.rows), dim3(256), 0, stream, v);
    return hipGetLastError();
}

}  // namespace atlas
