// verify_kernels.hip -- drafted tokens accepted or rejected against the
// target's probabilities, with given random numbers (speculative sampling).
// No counterpart in the reference, which decodes greedily one token a step.
//
// With p_t = softmax(target[b, t] / temperature) and q_t that of the draft
// model (or certainty: q_t = 1 at the drafted token), draft t of sequence b is
// accepted while accept[b, t] * q_t(x_t) < p_t(x_t).  At the first rejection a
// token is drawn from r = max(p - q, 0) (from p where that is nothing), after
// none from p of the row behind the last draft: the first i with
// r_0 + .. + r_i > sample[b] * (r_0 + .. + r_{V-1}).
// NaN logits have no mass; the mass of a row with +inf lies on its +inf.
//
// The drawn token is decided by a border between running sums of up to 2^18
// terms, which 32-bit sums move by far more than one term; probabilities and
// sums are in 64 bits throughout.
//
// Launches: every row's maximum and sum per slice of 1024 logits; with a draft
// model, the residual's sum per slice of the row that was rejected; one
// workgroup a sequence that finds the slice and the token in it.  The second
// and third decide for themselves what was accepted (of more than kFusedDrafts
// drafts a launch of its own does).  Where nothing is taken off p but the drafted token,
// the slices' sums are the first launch's.
#include "exp2_f64.hpp"
#include "launch.hpp"

#include <algorithm>
#include <limits>

namespace atlas {
namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / kWave;
// the draw itself is one workgroup's: its latency counts
constexpr int kPickThreads = 1024;
constexpr uint32_t kSlice = 1024;  // a wavefront's, 16 logits a lane
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr uint32_t kFusedDrafts = 16;

typedef f32x4 f32x4_row __attribute__((aligned(4)));

// A row's masses are e^{(x - top) * inv}, `scale` = 32 inv log2(e): 1 at the top,
// of an infinite one too, 0 in a row that has none.  With an infinite top that
// is the same about zero, for 0 at the top and -inf elsewhere.
__device__ __forceinline__ float about(float x, float top) {
    return top == __builtin_inff() ? (x == top ? 0.0f : -__builtin_inff()) : x;
}
__device__ __forceinline__ double finite(float top) { return __builtin_isinf(top) ? 0.0 : static_cast<double>(top); }
__device__ __forceinline__ double mass(float x, float top, double scale, const Exp2& exp2_of) {
    return exp2_of((static_cast<double>(about(x, top)) - finite(top)) * scale);
}

__device__ __forceinline__ double wave_inclusive_scan_f64(double v) {
    v += dpp_f64<0x111, 0xf, true>(v);  // row_shr 1, 2, 4, 8
    v += dpp_f64<0x112, 0xf, true>(v);
    v += dpp_f64<0x114, 0xf, true>(v);
    v += dpp_f64<0x118, 0xf, true>(v);
    v += dpp_f64<0x142, 0xa, false>(v);  // the rows before
    v += dpp_f64<0x143, 0xc, false>(v);
    return v;
}

// A slice's maximum and, relative to it, its sum.
struct SliceStat {
    double sum;
    float top;
    float unused;
};

// What was accepted, and the row that is drawn from.
struct Decision {
    double target_sum, draft_sum;
    float target_top, draft_top;
    uint32_t row;       // accepted drafts = the row of the target
    uint32_t rejected;  // a draft was rejected there
};

struct VerifyParams {
    VerifyDraftArgs s;
    double scale;             // 32 inv_temperature log2(e)
    SliceStat* target_stats;  // [sequence][drafts + 1][slices]
    SliceStat* draft_stats;   // [sequence][drafts][slices]
    double* slice_sums;       // [sequence][slices]
    Decision* decisions;      // [sequence], of launches that decide apart
    uint32_t slices, blocks;  // of a row; blocks of kVerifyWaves slices
};

__device__ __forceinline__ uint32_t drafts_of(const VerifyDraftArgs& s, uint32_t seq) {
    return s.draft_lengths ? min(s.draft_lengths[seq], s.drafts) : s.drafts;
}

// A lane's logits of a wavefront's slice, four at a time.
constexpr int kEach = kSlice / kWave;
__device__ __forceinline__ uint32_t slice_at(int i) { return (i / 4 * kWave + threadIdx.x % kWave) * 4 + i % 4; }
__device__ __forceinline__ void load_slice(const float* logits, uint32_t first, uint32_t vocab, float (&x)[kEach]) {
    if (first + kSlice <= vocab) {
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
            const f32x4 y = *reinterpret_cast<const f32x4_row*>(logits + first + slice_at(4 * i));
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = number_or_none(y[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t at = first + slice_at(i);
            x[i] = at < vocab ? number_or_none(logits[at]) : -__builtin_inff();
        }
    }
}

// A wavefront a slice of a row; rows of a sequence: targets, then drafts.  Bytes
// and exponentials add up: 384 rows of 262144 logits 98 to 107 us, 3.8 to 4.1
// TB/s.  Two to eight slices a wavefront, the next one's logits on their way:
// 94 to 107 us, and 37 to 56 where one slice takes 34 (640 rows of 50257).
__global__ __launch_bounds__(kVerifyThreads) void verify_stats_kernel(VerifyParams v) {
    __shared__ uint2 table[32];
    const VerifyDraftArgs& s = v.s;
    const uint32_t rows = s.drafts + 1 + (s.draft ? s.drafts : 0);
    const uint32_t seq = blockIdx.x / (v.blocks * rows);
    const uint32_t rest = blockIdx.x % (v.blocks * rows);
    uint32_t row = rest / v.blocks;
    const uint32_t slice = rest % v.blocks * kVerifyWaves + threadIdx.x / kWave;
    const uint32_t count = drafts_of(s, seq);
    const bool of_target = row <= s.drafts;
    if (!of_target) row -= s.drafts + 1;
    if (row > count || (!of_target && row == count)) return;
    const float* logits = of_target ? s.target + (static_cast<uint64_t>(seq) * (s.drafts + 1) + row) * s.vocab
                                    : s.draft + (static_cast<uint64_t>(seq) * s.drafts + row) * s.vocab;
    float x[kEach];
    load_slice(logits, min(slice, v.slices - 1) * kSlice, s.vocab, x);
    Exp2::fill(table);
    const Exp2 exp2_of(table);
    __syncthreads();
    if (slice >= v.slices) return;
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kEach; ++i) top = fmaxf(top, x[i]);
    top = wave_max_tree_f32(top);
    if (top == __builtin_inff()) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) x[i] = about(x[i], top);
    }
    const double zero = finite(top);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += exp2_of((static_cast<double>(x[i]) - zero) * v.scale);
    sum = wave_sum_f64(sum);
    SliceStat* out = of_target ? v.target_stats + (static_cast<uint64_t>(seq) * (s.drafts + 1) + row) * v.slices
                               : v.draft_stats + (static_cast<uint64_t>(seq) * s.drafts + row) * v.slices;
    if (threadIdx.x % kWave == 0) out[slice] = SliceStat{sum, top, 0.0f};
}

// A row's maximum and sum from its slices, by one wavefront; `first`: the
// lane's first of them, loaded before.
__device__ __forceinline__ SliceStat first_stat(const SliceStat* slices, uint32_t count) {
    const uint32_t lane = threadIdx.x % kWave;
    return lane < count ? slices[lane] : SliceStat{0.0, -__builtin_inff(), 0.0f};
}
__device__ __forceinline__ void row_stat(const SliceStat& first, const SliceStat* slices, uint32_t count, double scale,
                                         const Exp2& exp2_of, float& top, double& sum) {
    const uint32_t lane = threadIdx.x % kWave;
    top = first.top;
    for (uint32_t i = lane + kWave; i < count; i += kWave) top = fmaxf(top, slices[i].top);
    top = wave_max_tree_f32(top);
    sum = first.sum * mass(first.top, top, scale, exp2_of);
    for (uint32_t i = lane + kWave; i < count; i += kWave) sum += slices[i].sum * mass(slices[i].top, top, scale, exp2_of);
    sum = wave_sum_f64(sum);
}

// The decision of a sequence by a workgroup: the rows' sums by its wavefronts
// in turn, the drafts' tests by its threads.  The table is filled, and `d` can
// be read, behind the barriers here.
template <int THREADS, uint32_t MOST>
__device__ void decide(const VerifyParams& v, uint32_t seq, const Exp2& exp2_of, Decision& d) {
    constexpr uint32_t kWaves = THREADS / kWave;
    __shared__ double sums[2][MOST + 1];
    __shared__ float tops[2][MOST + 1];
    __shared__ uint32_t first_rejected;
    const VerifyDraftArgs& s = v.s;
    const uint32_t count = drafts_of(s, seq), rows = count + 1 + (s.draft ? count : 0);
    if (threadIdx.x == 0) first_rejected = count;
    __syncthreads();
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave));
    const auto stats_of = [&](uint32_t r) {
        return r <= count ? v.target_stats + (static_cast<uint64_t>(seq) * (s.drafts + 1) + r) * v.slices
                          : v.draft_stats + (static_cast<uint64_t>(seq) * s.drafts + r - count - 1) * v.slices;
    };
    // three rows' loads at a time: one after another their latency is most of
    // a small call
    for (uint32_t r0 = wave; r0 < rows; r0 += 3 * kWaves) {
        SliceStat first[3];
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i) first[i] = first_stat(stats_of(min(r0 + i * kWaves, rows - 1)), v.slices);
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i) {
            const uint32_t r = r0 + i * kWaves;
            if (r >= rows) break;
            float top;
            double sum;
            row_stat(first[i], stats_of(r), v.slices, v.scale, exp2_of, top, sum);
            if (threadIdx.x % kWave == 0) {
                sums[r > count][r <= count ? r : r - count - 1] = sum;
                tops[r > count][r <= count ? r : r - count - 1] = top;
            }
        }
    }
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < count; t += THREADS) {
        const uint64_t at = static_cast<uint64_t>(seq) * s.drafts + t;
        const uint32_t token = s.draft_tokens[at];
        double p = 0.0, q = s.draft ? 0.0 : 1.0;
        if (token < s.vocab) {
            const float x = number_or_none(s.target[(static_cast<uint64_t>(seq) * (s.drafts + 1) + t) * s.vocab + token]);
            if (sums[0][t] > 0.0) p = mass(x, tops[0][t], v.scale, exp2_of) / sums[0][t];
            if (s.draft && sums[1][t] > 0.0)
                q = mass(number_or_none(s.draft[at * s.vocab + token]), tops[1][t], v.scale, exp2_of) / sums[1][t];
        }
        if (!(static_cast<double>(s.accept_uniform[at]) * q < p)) atomicMin(&first_rejected, t);
    }
    __syncthreads();
    d.row = first_rejected;
    d.rejected = d.row < count;
    d.target_sum = sums[0][d.row];
    d.target_top = tops[0][d.row];
    d.draft_sum = s.draft && d.rejected ? sums[1][d.row] : 0.0;
    d.draft_top = s.draft && d.rejected ? tops[1][d.row] : 0.0f;
}

__global__ __launch_bounds__(kPickThreads) void verify_decide_kernel(VerifyParams v) {
    __shared__ uint2 table[32];
    Exp2::fill(table);
    const Exp2 exp2_of(table);
    Decision d;
    decide<kPickThreads, 1024>(v, blockIdx.x, exp2_of, d);
    if (threadIdx.x == 0) v.decisions[blockIdx.x] = d;
}

// The terms of a draw, of the row that the decision names.
struct Terms {
    const float* target;
    const float* draft;  // null: none, or certainty at `token`
    uint32_t token;
    double scale, target_scale, draft_scale;  // 1 / sum, or 0
    float target_top, draft_top;

    __device__ Terms(const VerifyParams& v, uint32_t seq, const Decision& d, bool residual) {
        const VerifyDraftArgs& s = v.s;
        target = s.target + (static_cast<uint64_t>(seq) * (s.drafts + 1) + d.row) * s.vocab;
        const bool minus = residual && d.rejected;
        const uint64_t at = static_cast<uint64_t>(seq) * s.drafts + d.row;
        draft = minus && s.draft ? s.draft + at * s.vocab : nullptr;
        token = minus && !s.draft ? s.draft_tokens[at] : kNoToken;
        scale = v.scale;
        target_top = d.target_top;
        draft_top = d.draft_top;
        target_scale = d.target_sum > 0.0 ? 1.0 / d.target_sum : 0.0;
        draft_scale = d.draft_sum > 0.0 ? 1.0 / d.draft_sum : 0.0;
    }
    __device__ double term(float x, float y, uint32_t at, const Exp2& exp2_of) const {
        const double p = mass(x, target_top, scale, exp2_of) * target_scale;
        if (!draft) return at == token ? 0.0 : p;
        const double q = mass(y, draft_top, scale, exp2_of) * draft_scale;
        return p > q ? p - q : 0.0;
    }
};

// A wavefront a slice (64 sequences, two rows of 262144 logits each: 32 us):
// the residual's sum there, of a sequence with a draft
// rejected (of others the slices' own sums serve).  FUSED: every workgroup
// decides for itself, and the first leaves the decision for the next launch.
template <bool FUSED>
__global__ __launch_bounds__(kVerifyThreads) void verify_residual_kernel(VerifyParams v) {
    __shared__ uint2 table[32];
    const uint32_t seq = blockIdx.x / v.blocks, block = blockIdx.x % v.blocks;
    const uint32_t slice = block * kVerifyWaves + threadIdx.x / kWave;
    Exp2::fill(table);
    const Exp2 exp2_of(table);
    Decision d;
    if (FUSED) {
        decide<kVerifyThreads, kFusedDrafts>(v, seq, exp2_of, d);
        if (block == 0 && threadIdx.x == 0) v.decisions[seq] = d;
    } else {
        d = v.decisions[seq];
        __syncthreads();
    }
    if (!d.rejected || slice >= v.slices) return;
    const Terms terms(v, seq, d, true);
    float x[kEach], y[kEach];
    load_slice(terms.target, slice * kSlice, v.s.vocab, x);
    load_slice(terms.draft, slice * kSlice, v.s.vocab, y);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += terms.term(x[i], y[i], slice * kSlice + slice_at(i), exp2_of);
    sum = wave_sum_f64(sum);
    if (threadIdx.x % kWave == 0) v.slice_sums[static_cast<uint64_t>(seq) * v.slices + slice] = sum;
}

// Of each thread's value, the sum of those before it and of all.
template <int THREADS>
__device__ __forceinline__ double block_before_f64(double v, double& all) {
    constexpr uint32_t kWaves = THREADS / kWave;
    __shared__ double wave_all[kWaves];
    const double upto = wave_inclusive_scan_f64(v);
    const uint32_t wave = threadIdx.x / kWave;
    __syncthreads();  // wave_all may still be read from a call before
    if (threadIdx.x % kWave == kWave - 1) wave_all[wave] = upto;
    __syncthreads();
    double before = 0.0;
    all = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w == wave) before = all;
        all += wave_all[w];
    }
    const double own = __shfl_up(upto, 1, kWave);
    return before + (threadIdx.x % kWave ? own : 0.0);
}

// The least `at` of the threads with a hit and the greatest `last` of those
// with mass, both in the threads' order: one lane of a wavefront asks (1024
// threads on one counter of LDS took 3 us).
__device__ __forceinline__ void first_and_last(bool hit, uint32_t at, bool mass, uint32_t last, uint32_t& first_hit,
                                               uint32_t& last_mass) {
    const uint32_t lane = threadIdx.x % kWave;
    const uint64_t hits = __builtin_amdgcn_ballot_w64(hit), some = __builtin_amdgcn_ballot_w64(mass);
    if (hits && lane == static_cast<uint32_t>(__builtin_ctzll(hits))) atomicMin(&first_hit, at);
    if (some && lane == 63u - static_cast<uint32_t>(__builtin_clzll(some))) atomicMax(&last_mass, last);
}

// One workgroup a sequence: the slice that holds the draw, the token in it,
// and the row of results (5.5 us for one sequence, 7.4 for 64: loads that wait for
// each other).  Rounding may leave the goal just past the last
// running sum: the last item with mass is then the one.
template <bool FUSED>
__global__ __launch_bounds__(kPickThreads) void verify_pick_kernel(VerifyParams v) {
    __shared__ uint2 table[32];
    __shared__ uint32_t first_hit, last_mass;
    __shared__ double shared_before;
    const VerifyDraftArgs& s = v.s;
    const uint32_t seq = blockIdx.x, tid = threadIdx.x;
    // what does not hang on the decision is asked for before it
    const double* sums = v.slice_sums + static_cast<uint64_t>(seq) * v.slices;
    const double my_sum = s.draft && tid < v.slices ? sums[tid] : 0.0;
    const uint32_t my_token = tid < s.drafts ? s.draft_tokens[static_cast<uint64_t>(seq) * s.drafts + tid] : kNoToken;
    const double uniform = s.sample_uniform[seq];
    Exp2::fill(table);
    const Exp2 exp2_of(table);
    Decision d;
    if (FUSED) {
        decide<kPickThreads, kFusedDrafts>(v, seq, exp2_of, d);
    } else {
        d = v.decisions[seq];
        __syncthreads();
    }
    const SliceStat* stats = v.target_stats + (static_cast<uint64_t>(seq) * (s.drafts + 1) + d.row) * v.slices;
    const double target_scale = d.target_sum > 0.0 ? 1.0 / d.target_sum : 0.0;

    // this thread's term of a slice
    static_assert(kPickThreads == kSlice, "a logit a thread");
    const auto term_of = [&](const Terms& terms, uint32_t slice) {
        const uint32_t at = slice * kSlice + tid;
        if (at >= s.vocab) return 0.0;
        return terms.term(number_or_none(terms.target[at]), terms.draft ? number_or_none(terms.draft[at]) : 0.0f, at, exp2_of);
    };
    // the slice that lost the token that was proposed with certainty
    uint32_t short_slice = kNoToken;
    double short_sum = 0.0;
    if (d.rejected && !s.draft) {
        const uint32_t token = s.draft_tokens[static_cast<uint64_t>(seq) * s.drafts + d.row];
        if (token < s.vocab) {
            short_slice = token / kSlice;
            (void)block_before_f64<kPickThreads>(term_of(Terms(v, seq, d, true), short_slice), short_sum);
        }
    }
    bool residual = true;
    const auto part = [&](uint32_t i) {
        if (residual && d.rejected && s.draft) return i == tid ? my_sum : sums[i];
        if (residual && i == short_slice) return short_sum;
        return stats[i].sum * mass(stats[i].top, d.target_top, v.scale, exp2_of) * target_scale;
    };
    // slices [begin, end) are this thread's
    const uint32_t each = (v.slices + kPickThreads - 1) / kPickThreads;
    const uint32_t begin = min(tid * each, v.slices), end = min(begin + each, v.slices);
    double total = 0.0, run = 0.0, one = 0.0;
    for (;;) {
        double sum = 0.0;
        for (uint32_t i = begin; i < end; ++i) sum += one = part(i);
        run = block_before_f64<kPickThreads>(sum, total);
        if (total > 0.0 || !residual) break;
        residual = false;  // nothing is left of p: draw from p itself
    }
    const double goal = uniform * total;
    if (tid == 0) {
        first_hit = kNoToken;
        last_mass = 0;
    }
    __syncthreads();
    uint32_t mine = kNoToken, last = kNoToken;
    double mine_before = 0.0, last_before = 0.0;
    for (uint32_t i = begin; i < end; ++i) {
        const double x = each == 1 ? one : part(i);
        if (x > 0.0) {
            last = i;
            last_before = run;
            if (mine == kNoToken && run + x > goal) {
                mine = i;
                mine_before = run;
            }
        }
        run += x;
    }
    first_and_last(mine != kNoToken, mine, last != kNoToken, last, first_hit, last_mass);
    __syncthreads();
    const bool hit = first_hit != kNoToken;
    const uint32_t slice = hit ? first_hit : last_mass;
    if (hit ? mine == slice : last == slice) shared_before = hit ? mine_before : last_before;
    __syncthreads();
    uint32_t drawn = kNoToken;
    if (total > 0.0) {
        const double rest = goal - shared_before;
        const double term = term_of(Terms(v, seq, d, residual), slice);
        double all;
        const double upto = block_before_f64<kPickThreads>(term, all) + term;  // its barriers stand between the uses of first_hit
        if (tid == 0) {
            first_hit = kNoToken;
            last_mass = 0;
        }
        __syncthreads();
        const uint32_t at = slice * kSlice + tid;
        first_and_last(term > 0.0 && upto > rest, at, term > 0.0, at, first_hit, last_mass);
        __syncthreads();
        drawn = first_hit != kNoToken ? first_hit : last_mass;
    }
    const uint64_t to = static_cast<uint64_t>(seq) * (s.drafts + 1);
    // at most as many drafts as threads, and one token more
    if (tid < s.drafts) s.tokens[to + tid] = tid < d.row ? my_token : (tid == d.row ? drawn : kNoToken);
    if (tid == 0) {
        s.tokens[to + s.drafts] = d.row == s.drafts ? drawn : kNoToken;
        s.accepted[seq] = d.row;
    }
}

uint64_t round256(uint64_t v) { return (v + 255) / 256 * 256; }

struct VerifyPlan {
    uint32_t slices;
    uint64_t target_bytes, draft_bytes, sum_bytes, decision_bytes;
    uint64_t total() const { return target_bytes + draft_bytes + sum_bytes + decision_bytes; }
};

VerifyPlan verify_plan(uint32_t sequences, uint32_t drafts, uint32_t vocab) {
    VerifyPlan p;
    p.slices = static_cast<uint32_t>((static_cast<uint64_t>(vocab) + kSlice - 1) / kSlice);
    const uint64_t per_row = static_cast<uint64_t>(sequences) * p.slices;
    p.target_bytes = round256(per_row * (drafts + 1) * sizeof(SliceStat));
    p.draft_bytes = round256(per_row * drafts * sizeof(SliceStat));
    p.sum_bytes = round256(per_row * sizeof(double));
    p.decision_bytes = round256(sequences * sizeof(Decision));
    return p;
}

template <typename K>
hipError_t launch(hipStream_t stream, K kernel, uint32_t blocks, const VerifyParams& v, uint32_t threads = kVerifyThreads) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, stream, v);
    return hipGetLastError();
}

}  // namespace

uint64_t verify_draft_workspace(uint32_t sequences, uint32_t drafts, uint32_t vocab) {
    return verify_plan(sequences, drafts, vocab).total();
}

hipError_t launch_verify_draft(hipStream_t stream, const VerifyDraftArgs& s) {
    const VerifyPlan p = verify_plan(s.sequences, s.drafts, s.vocab);
    uint8_t* ws = static_cast<uint8_t*>(s.workspace);
    // finite: 0 * inf at the largest logit would leave its row no mass
    const double scale = std::min(s.inv_temperature * 0x1.71547652b82fep+5, std::numeric_limits<double>::max());
    VerifyParams v{s,
                   scale,
                   reinterpret_cast<SliceStat*>(ws),
                   reinterpret_cast<SliceStat*>(ws + p.target_bytes),
                   reinterpret_cast<double*>(ws + p.target_bytes + p.draft_bytes),
                   reinterpret_cast<Decision*>(ws + p.target_bytes + p.draft_bytes + p.sum_bytes),
                   p.slices,
                   (p.slices + kVerifyWaves - 1) / kVerifyWaves};
    if (s.drafts == 0) v.s.draft = nullptr;
    const uint32_t rows = s.drafts + 1 + (v.s.draft ? s.drafts : 0);
    hipError_t e = launch(stream, verify_stats_kernel, v.blocks * rows * s.sequences, v);
    if (e != hipSuccess) return e;
    // Deciding in the launches that need it saves one; where those are many
    // workgroups, deciding so often costs more.  Residual of 1 x 12 slices fused
    // 8 us, apart 5 + 5; of 64 x 64 slices fused 41, apart 8 + 30.
    const uint32_t blocks = v.blocks * s.sequences;
    const bool fused = s.drafts <= kFusedDrafts && (v.s.draft ? blocks : s.sequences) <= 256;
    if (!fused && (e = launch(stream, verify_decide_kernel, s.sequences, v, kPickThreads)) != hipSuccess) return e;
    if (v.s.draft) {
        e = fused ? launch(stream, verify_residual_kernel<true>, blocks, v) : launch(stream, verify_residual_kernel<false>, blocks, v);
        if (e != hipSuccess) return e;
    }
    return fused && !v.s.draft ? launch(stream, verify_pick_kernel<true>, s.sequences, v, kPickThreads)
                               : launch(stream, verify_pick_kernel<false>, s.sequences, v, kPickThreads);
}

}  // namespace atlas
