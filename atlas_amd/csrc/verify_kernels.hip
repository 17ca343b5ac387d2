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
// Four launches: every row's maximum and sum per slice of 4096 logits; one
// wavefront a sequence that accepts and rejects; the residual's sum per slice of the
// row that was rejected; one workgroup a sequence that finds the slice and
// the token in it.
#include "device_common.hpp"
#include "launch.hpp"

namespace atlas {
namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / kWave;
constexpr uint32_t kSlice = 4096;
constexpr uint32_t kNoToken = 0xffffffffu;

typedef f32x4 f32x4_row __attribute__((aligned(4)));

__device__ __forceinline__ float number_or_none(float x) { return x != x ? -__builtin_inff() : x; }

// e^{(x - top) * inv}: 1 at the top (also of an infinite one), 0 in a row
// that has none.
__device__ __forceinline__ double mass(float x, float top, double inv) {
    const double e = exp((static_cast<double>(x) - static_cast<double>(top)) * inv);
    return top == -__builtin_inff() ? 0.0 : (x == top ? 1.0 : e);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

// A slice's maximum and, relative to it, its sum.
struct SliceStat {
    double sum;
    float top;
    float unused;
};

// What the first two launches leave for the others.
struct Decision {
    double target_sum, draft_sum;  // of the row that is drawn from
    float target_top, draft_top;
    uint32_t row;       // accepted drafts = the row of the target
    uint32_t rejected;  // a draft was rejected there
};

struct VerifyParams {
    VerifyDraftArgs s;
    SliceStat* target_stats;  // [sequence][drafts + 1][slices]
    SliceStat* draft_stats;   // [sequence][drafts][slices]
    double* slice_sums;       // [sequence][slices]
    Decision* decisions;      // [sequence]
    uint32_t slices;
};

__device__ __forceinline__ uint32_t drafts_of(const VerifyDraftArgs& s, uint32_t seq) {
    return s.draft_lengths ? min(s.draft_lengths[seq], s.drafts) : s.drafts;
}

// blockIdx.x: slice, blockIdx.y: row in a sequence (targets, then drafts),
// blockIdx.z: sequence.
__global__ __launch_bounds__(kVerifyThreads) void verify_stats_kernel(VerifyParams v) {
    __shared__ float wave_top[kVerifyWaves];
    __shared__ double wave_sum[kVerifyWaves];
    const VerifyDraftArgs& s = v.s;
    const uint32_t rows = s.drafts + 1 + (s.draft ? s.drafts : 0);
    const uint32_t seq = blockIdx.x / (v.slices * rows);
    const uint32_t rest = blockIdx.x % (v.slices * rows);
    uint32_t row = rest / v.slices;
    const uint32_t slice = rest % v.slices;
    const uint32_t count = drafts_of(s, seq);
    const bool of_target = row <= s.drafts;
    if (!of_target) row -= s.drafts + 1;
    if (row > count || (!of_target && row == count)) return;
    const float* logits = of_target ? s.target + (static_cast<uint64_t>(seq) * (s.drafts + 1) + row) * s.vocab
                                    : s.draft + (static_cast<uint64_t>(seq) * s.drafts + row) * s.vocab;
    const uint32_t first = slice * kSlice;
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    constexpr int kEach = kSlice / kVerifyThreads;
    float x[kEach];
    if (first + kSlice <= s.vocab) {
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
            const f32x4 y = __builtin_nontemporal_load(
                reinterpret_cast<const f32x4_row*>(logits + first + (i * kVerifyThreads + threadIdx.x) * 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = y[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t at = first + i * kVerifyThreads + threadIdx.x;
            x[i] = at < s.vocab ? logits[at] : -__builtin_inff();
        }
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        x[i] = number_or_none(x[i]);
        top = fmaxf(top, x[i]);
    }
    top = wave_max_tree_f32(top);
    if (lane == 0) wave_top[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += mass(x[i], top, s.inv_temperature);
    sum = wave_sum_f64(sum);
    if (lane == 0) wave_sum[wave] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    SliceStat* out = of_target ? v.target_stats + (static_cast<uint64_t>(seq) * (s.drafts + 1) + row) * v.slices
                               : v.draft_stats + (static_cast<uint64_t>(seq) * s.drafts + row) * v.slices;
    out[slice] = SliceStat{(wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]), top, 0.0f};
}

// A row's maximum and sum from its slices, by one wavefront.
__device__ __forceinline__ void row_stat(const SliceStat* slices, uint32_t count, double inv, float& top, double& sum) {
    const uint32_t lane = threadIdx.x % kWave;
    top = -__builtin_inff();
    for (uint32_t i = lane; i < count; i += kWave) top = fmaxf(top, slices[i].top);
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    sum = 0.0;
    for (uint32_t i = lane; i < count; i += kWave) sum += slices[i].sum * mass(slices[i].top, top, inv);
    sum = wave_sum_f64(sum);
}

// One wavefront a sequence.
__global__ __launch_bounds__(kWave) void verify_decide_kernel(VerifyParams v) {
    const VerifyDraftArgs& s = v.s;
    const uint32_t seq = blockIdx.x;
    const uint32_t count = drafts_of(s, seq);
    Decision d{};
    uint32_t t = 0;
    for (;; ++t) {
        row_stat(v.target_stats + (static_cast<uint64_t>(seq) * (s.drafts + 1) + t) * v.slices, v.slices, s.inv_temperature,
                 d.target_top, d.target_sum);
        if (t == count) break;
        const uint64_t at = static_cast<uint64_t>(seq) * s.drafts + t;
        const uint32_t token = s.draft_tokens[at];
        double p = 0.0, q = s.draft ? 0.0 : 1.0;
        if (s.draft) row_stat(v.draft_stats + at * v.slices, v.slices, s.inv_temperature, d.draft_top, d.draft_sum);
        if (token < s.vocab) {
            const float x = number_or_none(s.target[(static_cast<uint64_t>(seq) * (s.drafts + 1) + t) * s.vocab + token]);
            if (d.target_sum > 0.0) p = mass(x, d.target_top, s.inv_temperature) / d.target_sum;
            if (s.draft && d.draft_sum > 0.0)
                q = mass(number_or_none(s.draft[at * s.vocab + token]), d.draft_top, s.inv_temperature) / d.draft_sum;
        }
        if (!(static_cast<double>(s.accept_uniform[at]) * q < p)) {
            d.rejected = 1;
            break;
        }
    }
    d.row = t;
    if (threadIdx.x == 0) {
        v.decisions[seq] = d;
        s.accepted[seq] = t;
    }
}

// What a draw's terms are, of the row that the decision names.
struct Terms {
    const float* target;
    const float* draft;  // null: none, or certainty at `token`
    uint32_t token;
    double inv, target_scale, draft_scale;  // 1 / sum, or 0
    float target_top, draft_top;

    __device__ Terms(const VerifyParams& v, uint32_t seq, const Decision& d, bool residual) {
        const VerifyDraftArgs& s = v.s;
        target = s.target + (static_cast<uint64_t>(seq) * (s.drafts + 1) + d.row) * s.vocab;
        const bool minus = residual && d.rejected;
        const uint64_t at = static_cast<uint64_t>(seq) * s.drafts + d.row;
        draft = minus && s.draft ? s.draft + at * s.vocab : nullptr;
        token = minus && !s.draft ? s.draft_tokens[at] : kNoToken;
        inv = s.inv_temperature;
        target_top = d.target_top;
        draft_top = d.draft_top;
        target_scale = d.target_sum > 0.0 ? 1.0 / d.target_sum : 0.0;
        draft_scale = d.draft_sum > 0.0 ? 1.0 / d.draft_sum : 0.0;
    }
    __device__ double term(uint32_t i) const {
        const double p = mass(number_or_none(target[i]), target_top, inv) * target_scale;
        if (draft) {
            const double q = mass(number_or_none(draft[i]), draft_top, inv) * draft_scale;
            return p > q ? p - q : 0.0;
        }
        return i == token ? 0.0 : p;
    }
};

// blockIdx.x: slice of sequence blockIdx.x / slices; the sums of the residual.
__global__ __launch_bounds__(kVerifyThreads) void verify_residual_kernel(VerifyParams v) {
    __shared__ double wave_sum[kVerifyWaves];
    const uint32_t seq = blockIdx.x / v.slices, slice = blockIdx.x % v.slices;
    const Decision d = v.decisions[seq];
    const Terms terms(v, seq, d, true);
    const uint32_t first = slice * kSlice, last = min(first + kSlice, v.s.vocab);
    double sum = 0.0;
    for (uint32_t i = first + threadIdx.x; i < last; i += kVerifyThreads) sum += terms.term(i);
    sum = wave_sum_f64(sum);
    if (threadIdx.x % kWave == 0) wave_sum[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        v.slice_sums[static_cast<uint64_t>(seq) * v.slices + slice] = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
}

// One workgroup a sequence: the token, and the row of results.
__global__ __launch_bounds__(kVerifyThreads) void verify_pick_kernel(VerifyParams v) {
    __shared__ double before[kVerifyThreads];
    __shared__ uint32_t shared_slice;
    __shared__ double shared_goal;
    __shared__ int shared_residual;
    __shared__ uint32_t first_hit, last_positive;
    const VerifyDraftArgs& s = v.s;
    const uint32_t seq = blockIdx.x, tid = threadIdx.x;
    const Decision d = v.decisions[seq];
    const double* sums = v.slice_sums + static_cast<uint64_t>(seq) * v.slices;
    const SliceStat* stats = v.target_stats + (static_cast<uint64_t>(seq) * (s.drafts + 1) + d.row) * v.slices;
    const double scale = d.target_sum > 0.0 ? 1.0 / d.target_sum : 0.0;
    if (tid == 0) {
        double total = 0.0;
        for (uint32_t i = 0; i < v.slices; ++i) total += sums[i];
        const bool residual = total > 0.0;
        if (!residual)
            for (uint32_t i = 0; i < v.slices; ++i) total += stats[i].sum * mass(stats[i].top, d.target_top, s.inv_temperature) * scale;
        const double goal = static_cast<double>(s.sample_uniform[seq]) * total;
        double run = 0.0, at_last = 0.0;
        uint32_t slice = kNoToken;
        for (uint32_t i = 0; i < v.slices; ++i) {
            const double part = residual ? sums[i] : stats[i].sum * mass(stats[i].top, d.target_top, s.inv_temperature) * scale;
            if (part > 0.0) {
                slice = i;
                at_last = run;
                if (run + part > goal) break;
            }
            run += part;
        }
        shared_slice = slice;
        shared_goal = goal - at_last;
        shared_residual = residual;
        first_hit = kNoToken;
        last_positive = 0;
    }
    __syncthreads();
    const uint32_t slice = shared_slice;
    if (slice != kNoToken) {
        const Terms terms(v, seq, d, shared_residual != 0);
        constexpr int kEach = kSlice / kVerifyThreads;
        const uint32_t first = slice * kSlice + tid * kEach;
        double run[kEach];
        double sum = 0.0;
        uint32_t last = 0;
        bool any = false;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const double x = first + i < s.vocab ? terms.term(first + i) : 0.0;
            sum += x;
            run[i] = x > 0.0 ? sum : -1.0;
            if (x > 0.0) {
                last = first + i;
                any = true;
            }
        }
        before[tid] = sum;
        __syncthreads();
        double offset = 0.0;
        for (uint32_t i = 0; i < tid; ++i) offset += before[i];
        if (any) atomicMax(&last_positive, last);
        for (int i = kEach - 1; i >= 0; --i)
            if (run[i] >= 0.0 && offset + run[i] > shared_goal) atomicMin(&first_hit, first + i);
        __syncthreads();
    }
    const uint64_t at = static_cast<uint64_t>(seq) * (s.drafts + 1);
    for (uint32_t i = tid; i <= s.drafts; i += kVerifyThreads) {
        uint32_t token = kNoToken;
        if (i < d.row) token = s.draft_tokens[static_cast<uint64_t>(seq) * s.drafts + i];
        // rounding may leave the goal just past the slice's own running sum
        if (i == d.row && slice != kNoToken) token = first_hit != kNoToken ? first_hit : last_positive;
        s.tokens[at + i] = token;
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

}  // namespace

uint64_t verify_draft_workspace(uint32_t sequences, uint32_t drafts, uint32_t vocab) {
    return verify_plan(sequences, drafts, vocab).total();
}

hipError_t launch_verify_draft(hipStream_t stream, const VerifyDraftArgs& s) {
    const VerifyPlan p = verify_plan(s.sequences, s.drafts, s.vocab);
    uint8_t* ws = static_cast<uint8_t*>(s.workspace);
    VerifyParams v{s,
                   reinterpret_cast<SliceStat*>(ws),
                   reinterpret_cast<SliceStat*>(ws + p.target_bytes),
                   reinterpret_cast<double*>(ws + p.target_bytes + p.draft_bytes),
                   reinterpret_cast<Decision*>(ws + p.target_bytes + p.draft_bytes + p.sum_bytes),
                   p.slices};
    const uint32_t rows = s.drafts + 1 + (s.draft ? s.drafts : 0);
    hipLaunchKernelGGL(verify_stats_kernel, dim3(p.slices * rows * s.sequences), dim3(kVerifyThreads), 0, stream, v);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(verify_decide_kernel, dim3(s.sequences), dim3(kWave), 0, stream, v);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(verify_residual_kernel, dim3(p.slices * s.sequences), dim3(kVerifyThreads), 0, stream, v);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(verify_pick_kernel, dim3(s.sequences), dim3(kVerifyThreads), 0, stream, v);
    return hipGetLastError();
}

}  // namespace atlas
