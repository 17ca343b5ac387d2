// kv_evict_kernels.hip -- a batch's caches cut to a budget: a sequence longer
// than it keeps its most recent positions and, of the older ones, those that
// have drawn the most attention (the weights that the prefix attention adds
// up).  No counterpart in the reference, whose caches hold every position.
//
// With n = min(lengths[b], capacity), a sequence of n <= budget keeps all its
// positions.  Otherwise positions n - recent .. n - 1 stay, and the
// budget - recent largest weights of the first n - recent; of equal weights
// the lowest position, NaN below every number, -0 equal to +0.  Kept rows
// (both planes) and weights move to the front in their order.
//
// Two launches: one workgroup a sequence selects, then rows and weights move.
// The selection is a radix select over the weights' ordered bits, eight at a
// time, with the keys in registers, and one numbering of the kept positions
// in their order.
#include "device_common.hpp"
#include "launch.hpp"

namespace atlas {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;
constexpr uint32_t kNoPosition = 0xffffffffu;

// Larger weights have larger keys; NaN is 0, below -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
    uint32_t b = __float_as_uint(w);
    b = w == 0.0f ? 0u : b;
    const uint32_t ordered = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return w != w ? 0u : ordered;
}

// Of each wavefront's number, the sum of those of the wavefronts before it.
__device__ __forceinline__ uint32_t waves_before(uint32_t mine, uint32_t (&room)[kSelectWaves]) {
    const uint32_t wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) room[wave] = mine;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSelectWaves; ++w) before += w < wave ? room[w] : 0u;
    return before;
}

// Wavefront w has the positions from w * span on, KEYS to a lane (position
// w * span + 64 k + lane), so that order is wavefronts, then k, then lanes.
// KEYS = 0: longer sequences, whose keys are read anew by every pass.
// Histogram bins have 16 counters, one for every lane % 16: few exponents
// share most weights, and lanes that add to one counter go one by one (a
// sequence of 65536 in one counter a bin took 193 us; so 52, of 2048 4.3 to 5.0 us).
template <int KEYS>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(KvEvictArgs a) {
    __shared__ uint32_t bins[256][16];
    __shared__ uint32_t found[3];
    __shared__ uint32_t room[2][kSelectWaves];
    const uint32_t seq = blockIdx.x, tid = threadIdx.x;
    const uint32_t lane = tid % kWave;
    const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(tid / kWave));
    const float* weights = a.weights + static_cast<uint64_t>(seq) * a.capacity;
    uint32_t* kept = a.kept + static_cast<uint64_t>(seq) * a.budget;
    const uint32_t n = min(a.lengths[seq], a.capacity);
    __syncthreads();  // lengths_out may be lengths
    if (n <= a.budget) {
        for (uint32_t i = tid; i < a.budget; i += kSelectThreads) kept[i] = i < n ? i : kNoPosition;
        if (tid == 0) a.lengths_out[seq] = n;
        return;
    }
    if (tid == 0) a.lengths_out[seq] = a.budget;
    const uint32_t old = n - a.recent, heavy = a.budget - a.recent;
    const uint32_t steps = KEYS ? KEYS : (n + kSelectThreads - 1) / kSelectThreads;
    const uint32_t first = wave * steps * kWave + lane;
    // how many of this lane's positions are old, and there: comparing k with
    // them, each pass anew (the empty asm), keeps 64 positions and 64 masks out of
    // the registers, which the 64 keys fill (128, and 11 more in scratch)
    uint32_t mine_old = old > first ? (old - first + kWave - 1) / kWave : 0u;
    uint32_t mine_all = n > first ? (n - first + kWave - 1) / kWave : 0u;
    const auto key_at = [&](uint32_t k) {
        if (k >= mine_old) return 0xffffffffu;  // recent: above every weight
        return weight_key(weights[first + k * kWave]);
    };
    uint32_t held[KEYS ? KEYS : 1];
    if (KEYS) {
        // sixteen loads are on their way before the first key is made of them:
        // one behind the other 64 of them took 35 us
        constexpr int kAtOnce = KEYS && KEYS < 16 ? KEYS : 16;
#pragma unroll
        for (int k0 = 0; k0 < KEYS; k0 += kAtOnce) {
#pragma unroll
            for (int k = k0; k < k0 + kAtOnce; ++k)
                held[k] = __float_as_uint(weights[static_cast<uint32_t>(k) < mine_old ? first + k * kWave : 0u]);
#pragma unroll
            for (int k = k0; k < k0 + kAtOnce; ++k)
                held[k] = static_cast<uint32_t>(k) < mine_old ? weight_key(__uint_as_float(held[k])) : 0xffffffffu;
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // f(k, key) for every position first + 64 k of this lane, in order
    const auto each = [&](auto&& f) {
        if constexpr (KEYS != 0) {
            asm volatile("" : "+v"(mine_old), "+v"(mine_all));
#pragma unroll
            for (uint32_t k = 0; k < KEYS; ++k) f(k, held[k]);
        } else {
            for (uint32_t k = 0; k < steps; ++k) f(k, key_at(k));
        }
    };

    // the heavy-th largest key of the first `old`, and how many of the keys
    // equal to it stay
    uint32_t threshold = 0xffffffffu, equal = 0;
    bool split = false;  // some of the equal ones stay, some do not
    if (heavy) {
        uint32_t prefix = 0, mask = 0, need = heavy;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t i = tid; i < 256 * 16; i += kSelectThreads) (&bins[0][0])[i] = 0;
            __syncthreads();
            each([&](uint32_t k, uint32_t key) {
                if (k < mine_old && (key & mask) == prefix) atomicAdd(&bins[(key >> shift) & 255][lane % 16], 1u);
            });
            __syncthreads();
            // thread 4 i + j sums a quarter of bin i; then one wavefront finds
            // the bin, lane l having bins 255 - 4 l and below
            uint32_t part = 0;
            {
                const uint32_t* b = &bins[tid / 4][4 * (tid % 4)];
                part = b[0] + b[1] + b[2] + b[3];
            }
            part += __shfl_xor(part, 1, kWave);
            part += __shfl_xor(part, 2, kWave);
            __syncthreads();
            if (tid % 4 == 0) bins[tid / 4][0] = part;
            __syncthreads();
            if (wave == 0) {
                uint32_t c[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[j] = bins[255 - 4 * lane - j][0];
                    sum += c[j];
                }
                const uint32_t upto = wave_inclusive_scan_u32(sum);
                uint32_t above = upto - sum;
                // exactly one lane and bin: above < need <= above + count
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (above < need && need <= above + c[j]) {
                        found[0] = 255 - 4 * lane - j;
                        found[1] = need - above;
                        found[2] = c[j];
                    }
                    above += c[j];
                }
            }
            __syncthreads();
            prefix |= found[0] << shift;
            mask |= 255u << shift;
            need = found[1];
            // all that the bin holds stay: the lower bits decide nothing
            if (found[2] == need) break;
        }
        threshold = prefix;
        equal = need;
        split = found[2] != need;
    }

    const uint64_t below = (1ull << lane) - 1;
    if (!split) {
        uint32_t count = 0;
        each([&](uint32_t k, uint32_t key) { count += k < mine_all && key >= threshold; });
        count = wave_inclusive_scan_u32(count);
        uint32_t to = waves_before(readlane_u32(count, kWave - 1), room[0]);
        each([&](uint32_t k, uint32_t key) {
            const bool stay = k < mine_all && key >= threshold;
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(stay);
            if (stay) kept[to + __popcll(lanes & below)] = first + k * kWave;
            to += __popcll(lanes);
        });
        return;
    }
    // the equal ones are numbered, then the ones that stay
    uint32_t same_mine = 0;
    each([&](uint32_t k, uint32_t key) { same_mine += __popcll(__builtin_amdgcn_ballot_w64(k < mine_old && key == threshold)); });
    const uint32_t same_before = waves_before(same_mine, room[0]);
    const auto stays = [&](uint32_t k, uint32_t key, uint32_t& same_run) {
        const uint64_t same_lanes = __builtin_amdgcn_ballot_w64(k < mine_old && key == threshold);
        const bool stay = k < mine_all && (key > threshold || (key == threshold && same_run + __popcll(same_lanes & below) < equal));
        same_run += __popcll(same_lanes);
        return stay;
    };
    uint32_t stay_mine = 0, run = same_before;
    each([&](uint32_t k, uint32_t key) { stay_mine += __popcll(__builtin_amdgcn_ballot_w64(stays(k, key, run))); });
    uint32_t to = waves_before(stay_mine, room[1]);
    run = same_before;
    each([&](uint32_t k, uint32_t key) {
        const bool stay = stays(k, key, run);
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(stay);
        if (stay) kept[to + __popcll(lanes & below)] = first + k * kWave;
        to += __popcll(lanes);
    });
}

// Rows to another cache, a thread a unit of T at a time, and the weights as
// rows of one unit: blockIdx.y is a sequence and a plane, or its weights.  Bound
// by its bytes: 256 sequences keeping up to 512 rows of 1 KiB, 0.5 GB, 91 us,
// 5.5 TB/s read and written.
constexpr int kMoveThreads = 256;

template <typename T>
__global__ __launch_bounds__(kMoveThreads) void evict_copy_kernel(KvEvictArgs a, uint32_t units) {
    const uint32_t seq = blockIdx.y / 3, plane = blockIdx.y % 3;
    const uint64_t first = static_cast<uint64_t>(seq) * a.capacity;
    const uint32_t* kept = a.kept + static_cast<uint64_t>(seq) * a.budget;
    const uint32_t stride = gridDim.x * kMoveThreads, tid = blockIdx.x * kMoveThreads + threadIdx.x;
    if (plane == 2) {
        if (a.weights == a.weights_out) return;
        for (uint32_t row = tid; row < a.budget; row += stride) {
            const uint32_t from = kept[row];
            if (from != kNoPosition) a.weights_out[first + row] = a.weights[first + from];
        }
        return;
    }
    const uint64_t base = (plane ? static_cast<uint64_t>(a.sequences) * a.capacity : 0) + first;
    const uint64_t total = static_cast<uint64_t>(a.budget) * units;
    for (uint64_t i = tid; i < total; i += stride) {
        const uint32_t row = static_cast<uint32_t>(i / units), unit = static_cast<uint32_t>(i % units);
        const uint32_t from = kept[row];
        if (from == kNoPosition) return;
        const T v = __builtin_nontemporal_load(reinterpret_cast<const T*>(a.cache) + (base + from) * units + unit);
        __builtin_nontemporal_store(v, reinterpret_cast<T*>(a.cache_out) + (base + row) * units + unit);
    }
}

// Rows within their cache: a workgroup owns a column of units of one sequence
// and plane and walks its rows from the front, eight to a thread a step, each
// step's loads before its stores.  A row only moves towards the front, so what
// a step loads lies behind all that earlier ones store.  The barrier of each
// step bounds it: the 256 sequences above 59 us (a third of their rows stay
// where they are).
constexpr int kShiftThreads = 1024;
constexpr int kShiftRows = 8;

template <typename T>
__device__ __forceinline__ void shift_rows(T* rows, const uint32_t* kept, uint32_t budget, uint32_t units, uint32_t unit0,
                                           uint32_t column) {
    const uint32_t slots = kShiftThreads / column, slot = threadIdx.x / column, unit = unit0 + threadIdx.x % column;
    const bool active = slot < slots && unit < units;
    for (uint32_t row0 = 0; row0 < budget; row0 += slots * kShiftRows) {
        T v[kShiftRows];
        uint32_t from[kShiftRows];
#pragma unroll
        for (int i = 0; i < kShiftRows; ++i) {
            const uint32_t row = row0 + slot + i * slots;
            from[i] = active && row < budget ? kept[row] : kNoPosition;
            if (from[i] == row) from[i] = kNoPosition;  // stays where it is
        }
#pragma unroll
        for (int i = 0; i < kShiftRows; ++i)
            if (from[i] != kNoPosition) v[i] = rows[static_cast<uint64_t>(from[i]) * units + unit];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kShiftRows; ++i)
            if (from[i] != kNoPosition) rows[static_cast<uint64_t>(row0 + slot + i * slots) * units + unit] = v[i];
    }
}

template <typename T>
__global__ __launch_bounds__(kShiftThreads) void evict_shift_kernel(KvEvictArgs a, uint32_t units, uint32_t column) {
    const uint32_t seq = blockIdx.y >> 1;
    const uint64_t plane = (blockIdx.y & 1) ? static_cast<uint64_t>(a.sequences) * a.capacity : 0;
    const uint64_t first = plane + static_cast<uint64_t>(seq) * a.capacity;
    shift_rows(reinterpret_cast<T*>(a.cache_out) + first * units, a.kept + static_cast<uint64_t>(seq) * a.budget, a.budget, units,
               blockIdx.x * column, column);
}

__global__ __launch_bounds__(kShiftThreads) void evict_shift_weights_kernel(KvEvictArgs a) {
    shift_rows(a.weights_out + static_cast<uint64_t>(blockIdx.x) * a.capacity, a.kept + static_cast<uint64_t>(blockIdx.x) * a.budget,
               a.budget, 1u, 0u, 1u);
}

__global__ __launch_bounds__(kShiftThreads) void evict_copy_weights_kernel(KvEvictArgs a) {
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * a.capacity;
    for (uint32_t row = threadIdx.x; row < a.budget; row += kShiftThreads) {
        const uint32_t from = a.kept[static_cast<uint64_t>(blockIdx.x) * a.budget + row];
        if (from != kNoPosition) a.weights_out[first + row] = a.weights[first + from];
    }
}

// One launch covers up to 65535 / 3 sequences; the planes are found from
// sequences * capacity, so a launch past the first only shifts the bases.
template <typename T>
hipError_t launch_move(hipStream_t stream, const KvEvictArgs& a, bool in_place) {
    const uint32_t units = a.row_bytes / sizeof(T);
    constexpr uint32_t kMost = 21845;
    for (uint32_t s0 = 0; s0 < a.sequences; s0 += kMost) {
        KvEvictArgs b = a;
        const uint32_t count = a.sequences - s0 < kMost ? a.sequences - s0 : kMost;
        const uint64_t positions = static_cast<uint64_t>(s0) * a.capacity;
        b.cache = a.cache + positions * a.row_bytes;
        b.cache_out = a.cache_out + positions * a.row_bytes;
        b.weights = a.weights + positions;
        b.weights_out = a.weights_out + positions;
        b.kept = a.kept + static_cast<uint64_t>(s0) * a.budget;
        if (in_place) {
            // 256 bytes of a row to a workgroup, or 64 where those are too few for
            // the chip (8 sequences keeping 30000 rows of 1088 bytes 386 -> 279 us,
            // one keeping 1024 of 768 bytes 8.4 -> 4.6)
            uint32_t column = 256 / sizeof(T);
            while (column > 64 / sizeof(T) && (units + column - 1) / column * 2 * count < 256) column /= 2;
            if (column > units) column = units;
            hipLaunchKernelGGL((evict_shift_kernel<T>), dim3((units + column - 1) / column, 2 * count), dim3(kShiftThreads), 0,
                               stream, b, units, column);
        } else {
            const uint64_t blocks = (static_cast<uint64_t>(a.budget) * units + kMoveThreads * 4 - 1) / (kMoveThreads * 4);
            hipLaunchKernelGGL((evict_copy_kernel<T>), dim3(static_cast<uint32_t>(blocks < 4096 ? blocks : 4096), 3 * count),
                               dim3(kMoveThreads), 0, stream, b, units);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int KEYS>
void launch_select(hipStream_t stream, const KvEvictArgs& a) {
    hipLaunchKernelGGL(evict_select_kernel<KEYS>, dim3(a.sequences), dim3(kSelectThreads), 0, stream, a);
}

}  // namespace

hipError_t launch_kv_evict(hipStream_t stream, const KvEvictArgs& a) {
    const uint32_t keys = (a.capacity + kSelectThreads - 1) / kSelectThreads;
    if (keys <= 1)
        launch_select<1>(stream, a);
    else if (keys <= 2)
        launch_select<2>(stream, a);
    else if (keys <= 4)
        launch_select<4>(stream, a);
    else if (keys <= 8)
        launch_select<8>(stream, a);
    else if (keys <= 16)
        launch_select<16>(stream, a);
    else if (keys <= 32)
        launch_select<32>(stream, a);
    else if (keys <= 64)
        launch_select<64>(stream, a);
    else
        launch_select<0>(stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const bool in_place = a.cache == a.cache_out;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.cache) | reinterpret_cast<uintptr_t>(a.cache_out) | a.row_bytes;
    if (bits % 16 == 0)
        e = launch_move<u32x4_t>(stream, a, in_place);
    else if (bits % 8 == 0)
        e = launch_move<u32x2_t>(stream, a, in_place);
    else if (bits % 4 == 0)
        e = launch_move<uint32_t>(stream, a, in_place);
    else
        e = launch_move<uint16_t>(stream, a, in_place);
    if (e != hipSuccess) return e;
    // the copy launch takes weights that go elsewhere along
    if (a.weights == a.weights_out)
        hipLaunchKernelGGL(evict_shift_weights_kernel, dim3(a.sequences), dim3(kShiftThreads), 0, stream, a);
    else if (in_place)
        hipLaunchKernelGGL(evict_copy_weights_kernel, dim3(a.sequences), dim3(kShiftThreads), 0, stream, a);
    else
        return hipSuccess;
    return hipGetLastError();
}

}  // namespace atlas
