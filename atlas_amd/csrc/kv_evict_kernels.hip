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
// Two launches: one workgroup a sequence selects, then the rows move.  The
// selection is a radix select over the weights' ordered bits, eight at a time,
// and one pass in position order that numbers the kept ones.
#include "device_common.hpp"
#include "launch.hpp"

namespace atlas {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;
constexpr int kMoveThreads = 256;
constexpr uint32_t kNoPosition = 0xffffffffu;

// Larger weights have larger keys; NaN is 0, below -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
    uint32_t b = __float_as_uint(w);
    b = w == 0.0f ? 0u : b;
    const uint32_t ordered = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return w != w ? 0u : ordered;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(KvEvictArgs a) {
    __shared__ uint32_t bins[256];
    __shared__ uint32_t found[2];
    __shared__ uint32_t wave_kept[kSelectWaves], wave_equal[kSelectWaves];
    const uint32_t seq = blockIdx.x, tid = threadIdx.x;
    const uint32_t lane = tid % kWave, wave = tid / kWave;
    const uint64_t base = static_cast<uint64_t>(seq) * a.capacity;
    const float* weights = a.weights + base;
    float* weights_out = a.weights_out + base;
    uint32_t* kept = a.kept + static_cast<uint64_t>(seq) * a.budget;
    const uint32_t n = min(a.lengths[seq], a.capacity);
    __syncthreads();  // lengths_out may be lengths
    if (n <= a.budget) {
        for (uint32_t i = tid; i < a.budget; i += kSelectThreads) kept[i] = i < n ? i : kNoPosition;
        if (weights_out != weights)
            for (uint32_t i = tid; i < n; i += kSelectThreads) weights_out[i] = weights[i];
        if (tid == 0) a.lengths_out[seq] = n;
        return;
    }
    if (tid == 0) a.lengths_out[seq] = a.budget;
    const uint32_t old = n - a.recent, heavy = a.budget - a.recent;

    // the heavy-th largest key of the first `old`, and how many of the keys
    // equal to it stay
    uint32_t threshold = 0xffffffffu, equal = 0;
    if (heavy) {
        uint32_t prefix = 0, mask = 0, need = heavy;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t i = tid; i < 256; i += kSelectThreads) bins[i] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < old; i += kSelectThreads) {
                const uint32_t key = weight_key(weights[i]);
                if ((key & mask) == prefix) atomicAdd(&bins[(key >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t left = need, bin = 255;
                while (bins[bin] < left) left -= bins[bin--];
                found[0] = bin;
                found[1] = left;
            }
            __syncthreads();
            prefix |= found[0] << shift;
            mask |= 255u << shift;
            need = found[1];
            __syncthreads();
        }
        threshold = prefix;
        equal = need;
    }

    uint32_t kept_before = 0, equal_before = 0;
    for (uint32_t first = 0; first < n; first += kSelectThreads) {
        const uint32_t i = first + tid;
        const float w = i < n ? weights[i] : 0.0f;
        const uint32_t key = weight_key(w);
        const bool is_old = i < old;
        const bool same = heavy && is_old && key == threshold;
        const uint64_t same_lanes = __builtin_amdgcn_ballot_w64(same);
        const uint64_t below = (1ull << lane) - 1;
        if (lane == 0) wave_equal[wave] = __popcll(same_lanes);
        __syncthreads();
        uint32_t rank = equal_before + __popcll(same_lanes & below), same_all = 0;
        for (uint32_t w2 = 0; w2 < kSelectWaves; ++w2) {
            if (w2 < wave) rank += wave_equal[w2];
            same_all += wave_equal[w2];
        }
        const bool stay = i < n && (!is_old || (heavy && (key > threshold || (same && rank < equal))));
        const uint64_t stay_lanes = __builtin_amdgcn_ballot_w64(stay);
        if (lane == 0) wave_kept[wave] = __popcll(stay_lanes);
        __syncthreads();
        uint32_t at = kept_before + __popcll(stay_lanes & below), stay_all = 0;
        for (uint32_t w2 = 0; w2 < kSelectWaves; ++w2) {
            if (w2 < wave) at += wave_kept[w2];
            stay_all += wave_kept[w2];
        }
        if (stay) {
            kept[at] = i;
            weights_out[at] = w;  // at <= first of this step's reads
        }
        kept_before += stay_all;
        equal_before += same_all;
        __syncthreads();
    }
}

// Rows to another cache: a thread a unit of T.
template <typename T>
__global__ __launch_bounds__(kMoveThreads) void evict_copy_kernel(KvEvictArgs a, uint32_t units) {
    const uint32_t line = blockIdx.y;  // sequence and plane
    const uint32_t seq = line >> 1;
    const uint64_t plane = (line & 1) ? static_cast<uint64_t>(a.sequences) * a.capacity : 0;
    const uint64_t first = plane + static_cast<uint64_t>(seq) * a.capacity;
    const uint32_t* kept = a.kept + static_cast<uint64_t>(seq) * a.budget;
    const uint64_t total = static_cast<uint64_t>(a.budget) * units;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * kMoveThreads;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kMoveThreads + threadIdx.x; i < total; i += stride) {
        const uint32_t row = static_cast<uint32_t>(i / units), unit = static_cast<uint32_t>(i % units);
        const uint32_t from = kept[row];
        if (from == kNoPosition) return;
        reinterpret_cast<T*>(a.cache_out)[(first + row) * units + unit] =
            reinterpret_cast<const T*>(a.cache)[(first + from) * units + unit];
    }
}

// Rows within their cache: a workgroup owns a column of units of one sequence
// and plane and walks its rows from the front, each step's loads before its
// stores.  A row only moves towards the front, so no later step reads what an
// earlier one wrote.
template <typename T>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(KvEvictArgs a, uint32_t units, uint32_t column) {
    const uint32_t line = blockIdx.y;
    const uint32_t seq = line >> 1;
    const uint64_t plane = (line & 1) ? static_cast<uint64_t>(a.sequences) * a.capacity : 0;
    const uint64_t first = plane + static_cast<uint64_t>(seq) * a.capacity;
    const uint32_t* kept = a.kept + static_cast<uint64_t>(seq) * a.budget;
    T* cache = reinterpret_cast<T*>(a.cache_out);
    const uint32_t unit0 = blockIdx.x * column;
    const uint32_t wide = min(column, units - unit0);
    const uint32_t rows_a_step = kMoveThreads / column;
    const uint32_t row_of = threadIdx.x / column, unit = unit0 + threadIdx.x % column;
    const bool active = row_of < rows_a_step && threadIdx.x % column < wide;
    for (uint32_t row0 = 0; row0 < a.budget; row0 += rows_a_step) {
        const uint32_t row = row0 + row_of;
        uint32_t from = kNoPosition;
        if (active && row < a.budget) from = kept[row];
        T v{};
        const bool moves = from != kNoPosition && from != row;
        if (moves) v = cache[(first + from) * units + unit];
        __syncthreads();
        if (moves) cache[(first + row) * units + unit] = v;
        __syncthreads();
    }
}

template <typename T>
hipError_t launch_move(hipStream_t stream, const KvEvictArgs& a) {
    const uint32_t units = a.row_bytes / sizeof(T);
    const uint32_t lines_max = 65534;  // planes of whole sequences
    for (uint32_t s0 = 0; s0 < a.sequences; s0 += lines_max / 2) {
        // the planes are found from sequences * capacity, so a launch past the
        // first only shifts the sequence's base
        KvEvictArgs b = a;
        const uint32_t count = a.sequences - s0 < lines_max / 2 ? a.sequences - s0 : lines_max / 2;
        const uint64_t shift = static_cast<uint64_t>(s0) * a.capacity * a.row_bytes;
        b.cache = a.cache + shift;
        b.cache_out = a.cache_out + shift;
        b.kept = a.kept + static_cast<uint64_t>(s0) * a.budget;
        if (a.cache == a.cache_out) {
            const uint32_t column = units < 16 ? units : 16;
            hipLaunchKernelGGL((evict_move_kernel<T>), dim3((units + column - 1) / column, 2 * count), dim3(kMoveThreads),
                               0, stream, b, units, column);
        } else {
            const uint64_t blocks = (static_cast<uint64_t>(a.budget) * units + kMoveThreads * 4 - 1) / (kMoveThreads * 4);
            hipLaunchKernelGGL((evict_copy_kernel<T>), dim3(static_cast<uint32_t>(blocks < 4096 ? blocks : 4096), 2 * count),
                               dim3(kMoveThreads), 0, stream, b, units);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_kv_evict(hipStream_t stream, const KvEvictArgs& a) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(a.sequences), dim3(kSelectThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.cache) | reinterpret_cast<uintptr_t>(a.cache_out) | a.row_bytes;
    if (bits % 16 == 0) return launch_move<u32x4_t>(stream, a);
    if (bits % 8 == 0) return launch_move<u32x2_t>(stream, a);
    if (bits % 4 == 0) return launch_move<uint32_t>(stream, a);
    return launch_move<uint16_t>(stream, a);
}

}  // namespace atlas
